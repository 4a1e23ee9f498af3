// A paged KV cache for many requests: block tables and slot maps built on the
// GPU, RoPE + append by slot, and the commit of a draft tree's accepted path.

#include <limits.h>

#include <type_traits>

#include "b2a_common.cuh"

namespace b2a {
namespace paged {

constexpr int kMaxNodes = B2A_TREE_MAX_NODES;

// ---------------------------------------------------------------------------
// Block tables, slot map, positions (b2a_page_plan)
// ---------------------------------------------------------------------------
// All of it follows from three prefix sums over the requests (tokens, pages
// to take, pages to give back).  Every CTA forms them itself (a few
// microseconds for hundreds of requests, and no second launch), then writes
// its share: a warp per request for table entries and returned pages, a
// thread per 4 tokens for the slot map.  Pages taken come from the ring's
// head and pages given back go to its tail: the two regions do not meet
// while free and held pages together fit the ring, so CTAs need no order.
// Latency-bound: 64 requests with 513 tree nodes 7.7 us, 251 requests with 511K
// tokens 10.4 us (6.4 MB).
constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = kPlanThreads * 4;  // tokens of a CTA

struct Plan {
  const int *lens, *add, *parents, *held;
  int* table;
  long long table_stride;
  int* ring;
  const int* state;
  int *held_out, *state_out, *cu, *seq, *pos, *slot;
  int B, max_tokens, max_pages, page_shift, ring_size;
  bool whole;  // seq, pos and slot take 16-byte stores
};

// Tokens, pages wanted from the ring and pages given back of request b.
__device__ __forceinline__ void plan_request(const Plan& p, int b, int& n, int& need, int& back,
                                             bool& fits) {
  const int add = p.add[b], len = p.lens[b], held = p.held[b];
  const bool bad = len < 0 || held < 0 || held > p.max_pages;
  n = add < 0 ? 0 : min(add, p.max_tokens + 1);
  const long long want = (static_cast<long long>(len) + n + (1 << p.page_shift) - 1) >> p.page_shift;
  fits = add >= 0 && !bad && want <= p.max_pages;
  // (no tokens, no pages: the lens of a request that ended may still be there)
  need = fits && n > 0 ? max(0, static_cast<int>(want) - held) : 0;
  back = add < 0 && !bad ? held : 0;
  if (bad) set_dev_error(B2A_ERR_POSITION, b);
}

__device__ __forceinline__ int clamp_int(long long x) {
  return x > INT_MAX ? INT_MAX : static_cast<int>(x);
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const __grid_constant__ Plan p) {
  pdl_wait();
  extern __shared__ int psm[];
  int* s_cu = psm;               // [B + 1] tokens before request b
  int* s_need = s_cu + p.B + 1;  // [B + 1] pages taken before request b
  int* s_back = s_need + p.B + 1;  // [B + 1] pages given back before request b
  __shared__ long long s_part[3][kPlanThreads / 32];
  __shared__ long long s_run[3];
  __shared__ int s_par[kPlanTokens + kMaxNodes];
  __shared__ int s_taken;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kWarps = kPlanThreads / 32;
  const int gw = blockIdx.x * kWarps + warp, n_warps = gridDim.x * kWarps;
  // (kept inside the ring whatever the state holds)
  const int head = static_cast<int>(static_cast<unsigned>(p.state[0]) % static_cast<unsigned>(p.ring_size));
  const int count = min(max(p.state[1], 0), p.ring_size);
  if (tid < 3) s_run[tid] = 0;
  if (tid == 0) s_taken = 0;
  __syncthreads();
  // the prefix sums, kPlanThreads requests at a time
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int n = 0, need = 0, back = 0;
    bool fits = false;
    if (b < p.B) plan_request(p, b, n, need, back, fits);
    long long v[3] = {n, need, back}, inc[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      inc[k] = v[k];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc[k], o);
        if (lane >= o) inc[k] += x;
      }
      if (lane == 31) s_part[k][warp] = inc[k];
    }
    __syncthreads();
    long long before[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      before[k] = s_run[k];
      for (int w = 0; w < warp; ++w) before[k] += s_part[k][w];
      before[k] += inc[k] - v[k];
    }
    if (b < p.B) {
      s_cu[b] = clamp_int(before[0]);
      s_need[b] = clamp_int(before[1]);
      const long long upto = before[1] + need;
      const bool served = fits && (need == 0 || upto <= count);
      if (served && need > 0) atomicMax(&s_taken, static_cast<int>(upto));
      if (blockIdx.x == 0) {
        p.cu[b] = clamp_int(before[0]);
        p.held_out[b] = p.add[b] < 0 ? p.held[b] - back : p.held[b] + (served ? need : 0);
      }
      s_back[b] = clamp_int(before[2]);
    }
    __syncthreads();
    if (tid < 3) {
      long long t = s_run[tid];
      for (int w = 0; w < kWarps; ++w) t += s_part[tid][w];
      s_run[tid] = t;
    }
    __syncthreads();
  }
  const int total = clamp_int(s_run[0]);
  if (tid == 0) {
    s_cu[p.B] = total;
    s_need[p.B] = clamp_int(s_run[1]);
    s_back[p.B] = clamp_int(s_run[2]);
    if (blockIdx.x == 0) {
      p.cu[p.B] = total;
      p.state_out[0] = static_cast<int>((static_cast<long long>(head) + s_taken) % p.ring_size);
      p.state_out[1] = clamp_int(static_cast<long long>(count) - s_taken + s_run[2]);
      if (total > p.max_tokens) set_dev_error(B2A_ERR_POSITION, total);
    }
  }
  __syncthreads();
  // new table entries, and pages given back
  for (int b = gw; b < p.B; b += n_warps) {
    const int back = s_back[b + 1] - s_back[b];
    for (int j = lane; j < back; j += 32)
      p.ring[(static_cast<long long>(head) + count + s_back[b] + j) % p.ring_size] =
          p.table[b * p.table_stride + j];
    const int lo = s_need[b], need = s_need[b + 1] - lo;
    // a request that is not served has -1 where its pages would be: the entries
    // may hold pages of an earlier request that are others' by now
    const bool served = s_need[b + 1] <= count;
    const int held = need > 0 ? p.held[b] : 0;
    for (int k = lane; k < need; k += 32)
      p.table[b * p.table_stride + held + k] =
          served ? p.ring[(static_cast<long long>(head) + lo + k) % p.ring_size] : -1;
  }
  // tokens
  const int t0 = blockIdx.x * kPlanTokens;
  if (t0 >= p.max_tokens) return;
  auto find = [&](int t) {  // the request that holds token t < total
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_cu[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  int par0 = 0;
  if (p.parents && t0 < total) {
    // the tile's parents, from the first node of the tree that it cuts: at most
    // kMaxNodes before the tile (a tile of padding has none)
    const int end = min(min(t0 + kPlanTokens, p.max_tokens), total);
    par0 = max(s_cu[find(t0)], t0 - kMaxNodes);
    for (int i = tid; par0 + i < end; i += kPlanThreads) s_par[i] = p.parents[par0 + i];
    __syncthreads();
  }
  const int first = t0 + tid * 4;
  int b = first < total ? find(first) : 0;
  int sq[4], ps[4], sl[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int t = first + e;
    sq[e] = -1;
    ps[e] = 0;
    sl[e] = -1;
    if (t >= total || t >= p.max_tokens) continue;
    while (t >= s_cu[b + 1]) ++b;
    const int i = t - s_cu[b];
    const int len = p.lens[b], held = p.held[b];
    int depth = i;
    if (p.parents) {
      depth = 0;
      int at = i;
      const int base = s_cu[b] - par0;
      if (i >= kMaxNodes) {
        set_dev_error(B2A_ERR_POSITION, b);
      } else {
        while (true) {
          const int up = s_par[base + at];
          if (up < 0 || up >= at) {
            if (up != -1) set_dev_error(B2A_ERR_POSITION, b);
            break;
          }
          at = up;
          ++depth;
        }
      }
    }
    sq[e] = b;
    ps[e] = len + depth;
    const int lo = s_need[b], need = s_need[b + 1] - lo;
    int n_, need_, back_;
    bool fits;
    plan_request(p, b, n_, need_, back_, fits);
    if (fits && (need == 0 || s_need[b + 1] <= count)) {
      const int row = len + i, pg = row >> p.page_shift;
      const int page = pg < held ? p.table[b * p.table_stride + pg]
                                 : p.ring[(static_cast<long long>(head) + lo + pg - held) % p.ring_size];
      if (page < 0 || page > (INT_MAX >> p.page_shift)) {
        set_dev_error(B2A_ERR_POSITION, b);  // no page: its slot would be another's
      } else {
        sl[e] = (page << p.page_shift) + (row & ((1 << p.page_shift) - 1));
      }
    }
  }
  if (p.whole && first + 3 < p.max_tokens) {
    *reinterpret_cast<int4*>(p.seq + first) = make_int4(sq[0], sq[1], sq[2], sq[3]);
    *reinterpret_cast<int4*>(p.pos + first) = make_int4(ps[0], ps[1], ps[2], ps[3]);
    *reinterpret_cast<int4*>(p.slot + first) = make_int4(sl[0], sl[1], sl[2], sl[3]);
  } else {
    for (int e = 0; e < 4; ++e)
      if (first + e < p.max_tokens) {
        p.seq[first + e] = sq[e];
        p.pos[first + e] = ps[e];
        p.slot[first + e] = sl[e];
      }
  }
}

// ---------------------------------------------------------------------------
// RoPE + append by slot (b2a_rope_append_paged)
// ---------------------------------------------------------------------------
// Bound by reading the projections and writing q and the pool.  Products and
// sums are rounded one by one, as rope_append.cu does.  Two kernels:
//   rope_paged_rows   rows in 16-byte aligned groups of 8 elements.  A thread
//     keeps its 4 pairs' cosines and sines and goes over heads with them; the
//     loads of kHeads heads are in flight at once, before the position is known.
//     8 CTAs per SM go over the tokens (8191 tokens, 32/8 heads x 64, f16: 27.7 us;
//     a CTA per token 29.7; one pair per thread and step 83).
//   rope_paged_pairs  anything else (odd head or rotation widths, unaligned
//     strides): one pair per thread and step.
struct RopeArgs {
  const void *q, *k, *v;
  long long q_stride, k_stride, v_stride;
  const float *bq, *bk, *bv, *cos_tab, *sin_tab;
  const int *pos, *slots;
  void *k_pool, *v_pool, *q_out;
  long long page_stride, n_slots;
  int tab_rows, page_shift, H, KV, D, n_rot, neox, n_tok;
};

// The token's position and pool row (negative: not stored); false if the
// token is left out.
__device__ __forceinline__ bool rope_token(const RopeArgs& a, int i, int& p, long long& row) {
  p = a.pos[i];
  const int slot = a.slots[i];
  if (p < 0 || p >= a.tab_rows || slot >= a.n_slots) {
    if (threadIdx.x == 0 && blockIdx.y == 0) set_dev_error(B2A_ERR_POSITION, i);
    return false;
  }
  row = slot < 0 ? -1
                 : static_cast<long long>(slot >> a.page_shift) * a.page_stride +
                       static_cast<long long>(slot & ((1 << a.page_shift) - 1)) * a.KV * a.D;
  return true;
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = ld_elem(h + e);
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    load4(p, x);
    load4(p + 4, x + 4);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = ld_elem(h + e);
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(MmaOp<T>::pack(x[0], x[1]), MmaOp<T>::pack(x[2], x[3]));
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    store4(p, x);
    store4(p + 4, x + 4);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(MmaOp<T>::pack(x[0], x[1]), MmaOp<T>::pack(x[2], x[3]),
                                              MmaOp<T>::pack(x[4], x[5]), MmaOp<T>::pack(x[6], x[7]));
  }
}

constexpr int kRopeThreads = 256;
constexpr int kHeads = 3;  // heads of a thread with their loads in flight

template <typename TS, typename TK, typename TQ>
__global__ void __launch_bounds__(kRopeThreads) rope_paged_rows(const __grid_constant__ RopeArgs a) {
  pdl_wait();
  const int groups = a.D >> 3;              // groups of 8 elements (4 pairs) of a head
  const int heads_at_once = blockDim.x / groups;
  const int g = threadIdx.x % groups, h0 = threadIdx.x / groups;
  if (h0 >= heads_at_once) return;
  const int half = a.n_rot >> 1;
  const bool turned = 4 * g < half;         // the group's pairs rotate
  // elements of the group: [lo, lo + 4) and [hi, hi + 4)
  const bool split = a.neox && turned;
  const int lo = split ? 4 * g : 8 * g, hi = split ? half + 4 * g : 8 * g + 4;
  const int all = a.H + 2 * a.KV;
  const int step = heads_at_once * gridDim.y;
  for (int i = blockIdx.x; i < a.n_tok; i += gridDim.x) {
    float c[4], s[4];
    int p = -1;  // position, known once the first rows are on their way
    long long row = -1;
    for (int hb = blockIdx.y * heads_at_once + h0; hb < all; hb += kHeads * step) {
      float x[kHeads][8];
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int h = hb + u * step;
        if (h >= all) continue;
        const TS* src = h < a.H ? static_cast<const TS*>(a.q) + i * a.q_stride + h * a.D
                      : h < a.H + a.KV ? static_cast<const TS*>(a.k) + i * a.k_stride + (h - a.H) * a.D
                                       : static_cast<const TS*>(a.v) + i * a.v_stride + (h - a.H - a.KV) * a.D;
        if (split && h < a.H + a.KV) {
          load4(src + lo, x[u]);
          load4(src + hi, x[u] + 4);
        } else {
          load8(src + 8 * g, x[u]);
        }
      }
      if (p < 0) {
        if (!rope_token(a, i, p, row)) break;
        if (turned) {
          load4(a.cos_tab + static_cast<size_t>(p) * half + 4 * g, c);
          load4(a.sin_tab + static_cast<size_t>(p) * half + 4 * g, s);
        }
      }
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int h = hb + u * step;
        if (h >= all || (row < 0 && h >= a.H)) continue;
        const bool is_v = h >= a.H + a.KV;
        const bool part = split && !is_v;
        const float* bias = h < a.H ? a.bq : (is_v ? a.bv : a.bk);
        const int hh = h < a.H ? h : (is_v ? h - a.H - a.KV : h - a.H);
        const int la = part ? lo : 8 * g, ha = part ? hi : 8 * g + 4;
        if (bias) {
          float b[8];
          load4(bias + hh * a.D + la, b);
          load4(bias + hh * a.D + ha, b + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[u][e] = __fadd_rn(x[u][e], b[e]);
        }
        if (turned && !is_v) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x0 = a.neox ? x[u][e] : x[u][2 * e];
            const float x1 = a.neox ? x[u][e + 4] : x[u][2 * e + 1];
            const float y0 = __fsub_rn(__fmul_rn(x0, c[e]), __fmul_rn(x1, s[e]));
            const float y1 = __fadd_rn(__fmul_rn(x0, s[e]), __fmul_rn(x1, c[e]));
            if (a.neox) {
              x[u][e] = y0;
              x[u][e + 4] = y1;
            } else {
              x[u][2 * e] = y0;
              x[u][2 * e + 1] = y1;
            }
          }
        }
        if (h < a.H) {
          TQ* dst = static_cast<TQ*>(a.q_out) + (static_cast<size_t>(i) * a.H + h) * a.D;
          if (part) {
            store4(dst + lo, x[u]);
            store4(dst + hi, x[u] + 4);
          } else {
            store8(dst + 8 * g, x[u]);
          }
        } else {
          TK* dst = static_cast<TK*>(is_v ? a.v_pool : a.k_pool) + row + hh * a.D;
          if (part) {
            store4(dst + lo, x[u]);
            store4(dst + hi, x[u] + 4);
          } else {
            store8(dst + 8 * g, x[u]);
          }
        }
      }
    }
  }
}

template <typename TS, typename TK, typename TQ>
__global__ void __launch_bounds__(kRopeThreads) rope_paged_pairs(const __grid_constant__ RopeArgs a) {
  pdl_wait();
  const int i = blockIdx.x;
  int p;
  long long row;
  if (!rope_token(a, i, p, row)) return;
  const int half = a.n_rot >> 1, per = a.D >> 1;
  for (int u = blockIdx.y * kRopeThreads + threadIdx.x; u < (a.H + 2 * a.KV) * per;
       u += gridDim.y * kRopeThreads) {
    const int head = u / per, t = u - head * per;
    const bool is_q = head < a.H, is_v = head >= a.H + a.KV;
    const int h = is_q ? head : (is_v ? head - a.H - a.KV : head - a.H);
    if (!is_q && row < 0) continue;
    const TS* src = (is_q ? static_cast<const TS*>(a.q) + i * a.q_stride
                          : is_v ? static_cast<const TS*>(a.v) + i * a.v_stride
                                 : static_cast<const TS*>(a.k) + i * a.k_stride) + h * a.D;
    const float* bias = is_q ? a.bq : (is_v ? a.bv : a.bk);
    int e0 = 2 * t, e1 = 2 * t + 1;
    const bool turn = !is_v && t < half;
    if (turn && a.neox) {
      e0 = t;
      e1 = t + half;
    }
    float x0 = ld_elem(src + e0), x1 = ld_elem(src + e1);
    if (bias) {
      x0 = __fadd_rn(x0, bias[h * a.D + e0]);
      x1 = __fadd_rn(x1, bias[h * a.D + e1]);
    }
    float y0 = x0, y1 = x1;
    if (turn) {
      const float c = a.cos_tab[static_cast<size_t>(p) * half + t];
      const float s = a.sin_tab[static_cast<size_t>(p) * half + t];
      y0 = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
      y1 = __fadd_rn(__fmul_rn(x0, s), __fmul_rn(x1, c));
    }
    if (is_q) {
      TQ* dst = static_cast<TQ*>(a.q_out) + (static_cast<size_t>(i) * a.H + h) * a.D;
      st_elem(dst + e0, y0);
      st_elem(dst + e1, y1);
    } else {
      TK* dst = static_cast<TK*>(is_v ? a.v_pool : a.k_pool) + row + h * a.D;
      st_elem(dst + e0, y0);
      st_elem(dst + e1, y1);
    }
  }
}

// ---------------------------------------------------------------------------
// Accepted path and row moves (b2a_tree_commit)
// ---------------------------------------------------------------------------
// From the root, the path goes on to the first child whose token is the
// node's pick (-1, nothing to pick, ends it).  A request that the plan did not serve (its last row has no page)
// has no path.  Warp 0 of every CTA walks it (each step is one ballot over
// the request's nodes), then each thread moves one 16-byte column of the
// path's rows, in path order: the row at depth d comes from node path[d] >= d,
// so no row is overwritten before it was read.  Latency-bound: 16 layers, one
// request 4.1 us.
constexpr int kCommitThreads = 256;

struct Commit {
  const int *picks, *tokens, *parents, *cu, *lens, *table;
  long long table_stride;
  unsigned char *k, *v;
  long long layer_bytes, page_bytes;
  int row_bytes, n_layers, n_pages, page_shift;  // page_shift < 0: one block per sequence
  int max_len, n_tok, max_nodes;
  int *path, *accepted, *next, *lens_out;
};

__global__ void __launch_bounds__(kCommitThreads) tree_commit_kernel(const __grid_constant__ Commit c) {
  pdl_wait();
  __shared__ int s_path[kMaxNodes];
  __shared__ long long s_src[kMaxNodes], s_dst[kMaxNodes];
  __shared__ int s_n;
  const int b = blockIdx.y;
  const int lane = threadIdx.x & 31;
  const int c0 = c.cu[b], n = c.cu[b + 1] - c0, len = c.lens[b];
  const bool bad = n < 0 || n > c.max_nodes || c0 < 0 || c0 + n > c.n_tok || len < 0 ||
                   len > c.max_len - n;
  const bool served = !bad && n > 0 &&
                      (c.page_shift < 0 ||
                       c.table[b * c.table_stride + ((len + n - 1) >> c.page_shift)] != -1);
  if (threadIdx.x < 32) {
    int par[kMaxNodes / 32], tok[kMaxNodes / 32], pick[kMaxNodes / 32];
#pragma unroll
    for (int w = 0; w < kMaxNodes / 32; ++w) {
      const int j = w * 32 + lane;
      const bool in = served && j < n;
      par[w] = in ? (c.parents ? c.parents[c0 + j] : j - 1) : -2;
      tok[w] = in ? c.tokens[c0 + j] : 0;
      pick[w] = in ? c.picks[c0 + j] : 0;
    }
    int len_path = 0, cur = 0, last = -1;
    if (served) {
      while (true) {
        if (lane == 0) s_path[len_path] = cur;
        ++len_path;
#pragma unroll
        for (int w = 0; w < kMaxNodes / 32; ++w)
          if (w == cur >> 5) last = __shfl_sync(0xffffffffu, pick[w], cur & 31);
        int nxt = -1;
#pragma unroll
        for (int w = 0; w < kMaxNodes / 32; ++w) {
          const int j = w * 32 + lane;
          const unsigned hit =
              __ballot_sync(0xffffffffu, last >= 0 && par[w] == cur && j > cur && tok[w] == last);
          if (nxt < 0 && hit) nxt = w * 32 + __ffs(hit) - 1;
        }
        if (nxt < 0) break;
        cur = nxt;
      }
    }
    __syncwarp();
    if (blockIdx.x == 0) {
      for (int d = lane; d < c.max_nodes; d += 32)
        c.path[static_cast<size_t>(b) * c.max_nodes + d] = d < len_path ? s_path[d] : -1;
      if (lane == 0) {
        c.accepted[b] = len_path;
        c.next[b] = last;
        c.lens_out[b] = len + len_path;
        if (bad) set_dev_error(B2A_ERR_POSITION, b);
      }
    }
    for (int d = lane; d < len_path; d += 32) {
      const int from = len + s_path[d], to = len + d;
      long long src = -1, dst = -1;
      if (from != to) {
        if (c.page_shift < 0) {
          src = b * c.page_bytes + static_cast<long long>(from) * c.row_bytes;
          dst = b * c.page_bytes + static_cast<long long>(to) * c.row_bytes;
        } else {
          const int pf = c.table[b * c.table_stride + (from >> c.page_shift)];
          const int pt = c.table[b * c.table_stride + (to >> c.page_shift)];
          const int mask = (1 << c.page_shift) - 1;
          if (pf < 0 || pf >= c.n_pages || pt < 0 || pt >= c.n_pages) {
            set_dev_error(B2A_ERR_POSITION, b);
          } else {
            src = pf * c.page_bytes + static_cast<long long>(from & mask) * c.row_bytes;
            dst = pt * c.page_bytes + static_cast<long long>(to & mask) * c.row_bytes;
          }
        }
      }
      s_src[d] = src;
      s_dst[d] = dst;
    }
    if (lane == 0) s_n = len_path;
  }
  __syncthreads();
  const int m = s_n;
  const int chunks = c.row_bytes >> 4;
  const int cols = c.n_layers * 2 * chunks;
  for (int u = blockIdx.x * kCommitThreads + threadIdx.x; u < cols; u += gridDim.x * kCommitThreads) {
    const int row = u / chunks, at = u - row * chunks;
    unsigned char* base = ((row & 1) ? c.v : c.k) + (row >> 1) * c.layer_bytes + at * 16;
    for (int d = 0; d < m; ++d) {
      if (s_src[d] < 0) continue;
      const uint4 x = *reinterpret_cast<const uint4*>(base + s_src[d]);
      *reinterpret_cast<uint4*>(base + s_dst[d]) = x;
    }
  }
}

}  // namespace paged
}  // namespace b2a

// ===========================================================================
// Host side
// ===========================================================================
namespace {

namespace PG = b2a::paged;

template <typename TS, typename TK, typename TQ>
cudaError_t rope_paged_launch(const PG::RopeArgs& a, int n_tok, cudaStream_t st) {
  auto aligned = [](const void* p, long long stride, size_t es) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * static_cast<long long>(es) % 16 == 0;
  };
  const bool rows = a.D % 8 == 0 && a.n_rot % 8 == 0 && aligned(a.q, a.q_stride, sizeof(TS)) &&
                    aligned(a.k, a.k_stride, sizeof(TS)) && aligned(a.v, a.v_stride, sizeof(TS)) &&
                    aligned(a.q_out, 0, 2) && aligned(a.k_pool, a.page_stride, sizeof(TK)) &&
                    aligned(a.v_pool, 0, 2) && aligned(a.cos_tab, 0, 4) && aligned(a.sin_tab, 0, 4) &&
                    aligned(a.bq, 0, 4) && aligned(a.bk, 0, 4) && aligned(a.bv, 0, 4);
  const int all = a.H + 2 * a.KV;
  if (rows) {
    // as many threads as give each kHeads heads; few tokens: a token's heads
    // over more CTAs, until there are a few per SM
    const int groups = a.D / 8;
    int threads = ((all + PG::kHeads - 1) / PG::kHeads * groups + 31) / 32 * 32;
    if (threads > PG::kRopeThreads) threads = PG::kRopeThreads;
    int gy = (all + threads / groups - 1) / (threads / groups);
    const int enough = (4 * b2a_host::sm_count() + n_tok - 1) / n_tok;
    if (gy > enough) gy = enough;
    const int resident = 8 * b2a_host::sm_count();
    return b2a_host::launch(PG::rope_paged_rows<TS, TK, TQ>, dim3(n_tok < resident ? n_tok : resident, gy),
                            dim3(threads), 0, st, a);
  }
  const int pairs = all * (a.D / 2);
  return b2a_host::launch(PG::rope_paged_pairs<TS, TK, TQ>,
                          dim3(n_tok, (pairs + PG::kRopeThreads - 1) / PG::kRopeThreads),
                          dim3(PG::kRopeThreads), 0, st, a);
}

// Calls f with a null pointer of the element type of a dtype code.
template <typename F>
auto with_type(int dtype, F&& f) {
  if (dtype == B2A_F16) return f(static_cast<__half*>(nullptr));
  if (dtype == B2A_BF16) return f(static_cast<__nv_bfloat16*>(nullptr));
  return f(static_cast<float*>(nullptr));
}

}  // namespace

extern "C" {

int b2a_page_plan(const int* lens_dev, const int* add_dev, const int* parents_dev,
                  const int* held_dev, int* held_out_dev, int* table_dev, long long table_stride,
                  int* ring_dev, int ring_size, const int* ring_state_dev,
                  int* ring_state_out_dev, int* cu_dev, int* seq_dev, int* pos_dev, int* slot_dev,
                  int B, int max_tokens, int max_pages, int page_rows, void* stream) {
  if (!lens_dev || !add_dev || !held_dev || !held_out_dev || !table_dev || !ring_dev ||
      !ring_state_dev || !ring_state_out_dev || !cu_dev ||
      (max_tokens > 0 && (!seq_dev || !pos_dev || !slot_dev)))
    return fail(B2A_ERR_ARG, "page_plan: null pointer argument");
  if (B <= 0 || max_tokens < 0 || max_pages <= 0 || ring_size <= 0)
    return fail(B2A_ERR_ARG, "page_plan: sizes must be positive (B=%d max_tokens=%d max_pages=%d ring=%d)",
                B, max_tokens, max_pages, ring_size);
  if (B > B2A_PLAN_MAX_REQUESTS)
    return fail(B2A_ERR_UNSUPPORTED, "page_plan: %d requests > %d", B, B2A_PLAN_MAX_REQUESTS);
  if (!power_of_two(page_rows))
    return fail(B2A_ERR_SHAPE, "page_plan: page_rows %d is not a power of two", page_rows);
  if (table_stride < max_pages)
    return fail(B2A_ERR_SHAPE, "page_plan: table_stride %lld < max_pages %d", table_stride, max_pages);
  if (held_dev == held_out_dev || ring_state_dev == ring_state_out_dev)
    return fail(B2A_ERR_ARG, "page_plan: held and ring_state need output buffers of their own");
  if (static_cast<long long>(ring_size) * page_rows > INT_MAX)
    return fail(B2A_ERR_UNSUPPORTED, "page_plan: %d pages of %d rows exceed 32-bit slots", ring_size, page_rows);
  PG::Plan p = {lens_dev, add_dev, parents_dev, held_dev, table_dev, table_stride, ring_dev,
                ring_state_dev, held_out_dev, ring_state_out_dev, cu_dev, seq_dev, pos_dev,
                slot_dev, B, max_tokens, max_pages, log2_of(page_rows), ring_size,
                b2a_host::aligned16(seq_dev) && b2a_host::aligned16(pos_dev) && b2a_host::aligned16(slot_dev)};
  constexpr int kWarps = PG::kPlanThreads / 32;
  int grid = (max_tokens + PG::kPlanTokens - 1) / PG::kPlanTokens;
  if (grid < (B + kWarps - 1) / kWarps) grid = (B + kWarps - 1) / kWarps;
  const int smem = 3 * (B + 1) * static_cast<int>(sizeof(int));
  const cudaError_t e = b2a_host::launch(PG::page_plan_kernel, dim3(grid), dim3(PG::kPlanThreads),
                                         smem, static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "page_plan launch");
}

int b2a_rope_append_paged(const void* q, long long q_tok_stride, const void* k,
                          long long k_tok_stride, const void* v, long long v_tok_stride,
                          int in_dtype, const float* bq, const float* bk, const float* bv,
                          const float* cos_tab, const float* sin_tab, int tab_rows,
                          const int* pos_dev, const int* slot_dev, void* k_pool, void* v_pool,
                          int n_pages, int page_rows, long long page_stride, int kv_dtype,
                          void* q_out, int q_out_dtype, int n_tok, int H, int KV, int D, int n_rot,
                          int style, void* stream) {
  if (!q || !k || !v || !cos_tab || !sin_tab || !pos_dev || !slot_dev || !k_pool || !v_pool || !q_out)
    return fail(B2A_ERR_ARG, "rope_append_paged: null pointer argument");
  if (n_tok < 0 || H <= 0 || KV <= 0 || D <= 0 || tab_rows <= 0 || n_pages <= 0)
    return fail(B2A_ERR_ARG, "rope_append_paged: sizes must be positive (n_tok=%d H=%d KV=%d D=%d)",
                n_tok, H, KV, D);
  if (D % 2 != 0 || D > 256) return fail(B2A_ERR_UNSUPPORTED, "rope_append_paged: head_dim %d", D);
  if (n_rot < 0 || n_rot % 2 != 0 || n_rot > D)
    return fail(B2A_ERR_SHAPE, "rope_append_paged: n_rot %d (even, at most D=%d)", n_rot, D);
  if (style != B2A_ROPE_NORM && style != B2A_ROPE_NEOX)
    return fail(B2A_ERR_ARG, "rope_append_paged: style %d", style);
  const int es = b2a_host::elem_size(in_dtype);
  if (es == 0 || b2a_host::elem_size(kv_dtype) == 0 || b2a_host::elem_size(q_out_dtype) == 0)
    return fail(B2A_ERR_DTYPE, "rope_append_paged: dtypes %d, %d, %d", in_dtype, kv_dtype, q_out_dtype);
  if (!power_of_two(page_rows))
    return fail(B2A_ERR_SHAPE, "rope_append_paged: page_rows %d is not a power of two", page_rows);
  const long long page_elems = static_cast<long long>(page_rows) * KV * D;
  if (page_stride == 0) page_stride = page_elems;
  if (page_stride < page_elems)
    return fail(B2A_ERR_SHAPE, "rope_append_paged: page_stride %lld < page_rows*KV*D %lld", page_stride, page_elems);
  if (q_tok_stride < static_cast<long long>(H) * D || k_tok_stride < static_cast<long long>(KV) * D ||
      v_tok_stride < static_cast<long long>(KV) * D)
    return fail(B2A_ERR_SHAPE, "rope_append_paged: token strides overlap the rows");
  if (n_tok == 0) return B2A_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const PG::RopeArgs a = {q, k, v, q_tok_stride, k_tok_stride, v_tok_stride, bq, bk, bv, cos_tab,
                          sin_tab, pos_dev, slot_dev, k_pool, v_pool, q_out, page_stride,
                          static_cast<long long>(n_pages) * page_rows, tab_rows,
                          log2_of(page_rows), H, KV, D, n_rot, style == B2A_ROPE_NEOX ? 1 : 0, n_tok};
  const cudaError_t e = with_type(in_dtype, [&](auto* ts) {
    return with_type(kv_dtype, [&](auto* tk) {
      return with_type(q_out_dtype, [&](auto* tq) {
        using TS = typename std::remove_pointer<decltype(ts)>::type;
        using TK = typename std::remove_pointer<decltype(tk)>::type;
        using TQ = typename std::remove_pointer<decltype(tq)>::type;
        return rope_paged_launch<TS, TK, TQ>(a, n_tok, st);
      });
    });
  });
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "rope_append_paged launch");
}

int b2a_tree_commit(const int* picks_dev, const int* tokens_dev, const int* parents_dev,
                    const int* cu_dev, const int* lens_dev, const int* table_dev,
                    long long table_stride, int table_width, void* k_cache, void* v_cache,
                    int n_layers, long long layer_stride, int n_pages, int page_rows,
                    long long page_stride, int KV, int D, int dtype, int B, int n_tok,
                    int max_nodes, int max_len, int* path_dev, int* accepted_dev, int* next_dev,
                    int* lens_out_dev, void* stream) {
  if ((n_tok > 0 && (!picks_dev || !tokens_dev)) || !cu_dev || !lens_dev || !k_cache || !v_cache || !path_dev ||
      !accepted_dev || !next_dev || !lens_out_dev)
    return fail(B2A_ERR_ARG, "tree_commit: null pointer argument");
  if (n_layers <= 0 || n_pages <= 0 || page_rows <= 0 || KV <= 0 || D <= 0 || B <= 0 || n_tok < 0 || max_len <= 0)
    return fail(B2A_ERR_ARG, "tree_commit: sizes must be positive");
  if (max_nodes <= 0 || max_nodes > B2A_TREE_MAX_NODES)
    return fail(B2A_ERR_ARG, "tree_commit: max_nodes %d (1..%d)", max_nodes, B2A_TREE_MAX_NODES);
  if (B > 65535) return fail(B2A_ERR_UNSUPPORTED, "tree_commit: %d requests > 65535", B);
  if (lens_out_dev == lens_dev)
    return fail(B2A_ERR_ARG, "tree_commit: lens_out needs a buffer of its own");
  const int es = b2a_host::elem_size(dtype);
  if (es == 0) return fail(B2A_ERR_DTYPE, "tree_commit: dtype %d", dtype);
  const long long page_elems = static_cast<long long>(page_rows) * KV * D;
  if (page_stride == 0) page_stride = page_elems;
  if (page_stride < page_elems || (n_layers > 1 && layer_stride < page_stride * (n_pages - 1) + page_elems))
    return fail(B2A_ERR_SHAPE, "tree_commit: page or layer strides overlap");
  if (table_dev) {
    if (!power_of_two(page_rows))
      return fail(B2A_ERR_SHAPE, "tree_commit: page_rows %d is not a power of two", page_rows);
    if (table_width <= 0 || table_stride < table_width ||
        static_cast<long long>(table_width) * page_rows < max_len)
      return fail(B2A_ERR_SHAPE, "tree_commit: a table row of %d pages (stride %lld) does not hold max_len %d rows",
                  table_width, table_stride, max_len);
  } else if (n_pages < B || page_rows < max_len) {
    return fail(B2A_ERR_SHAPE, "tree_commit: %d blocks of %d rows for %d sequences of up to %d",
                n_pages, page_rows, B, max_len);
  }
  const long long row_bytes = static_cast<long long>(KV) * D * es;
  if (!b2a_host::aligned16(k_cache) || !b2a_host::aligned16(v_cache) || row_bytes % 16 != 0 ||
      (page_stride * es) % 16 != 0 || (n_layers > 1 && (layer_stride * es) % 16 != 0))
    return fail(B2A_ERR_ALIGN, "tree_commit: caches, rows and strides must be 16-byte aligned");
  PG::Commit c = {picks_dev, tokens_dev, parents_dev, cu_dev, lens_dev, table_dev, table_stride,
                  static_cast<unsigned char*>(k_cache), static_cast<unsigned char*>(v_cache),
                  n_layers > 1 ? layer_stride * es : 0, page_stride * es, static_cast<int>(row_bytes),
                  n_layers, n_pages, table_dev ? log2_of(page_rows) : -1, max_len, n_tok, max_nodes,
                  path_dev, accepted_dev, next_dev, lens_out_dev};
  const long long cols = static_cast<long long>(n_layers) * 2 * (row_bytes / 16);
  const long long gx = (cols + PG::kCommitThreads - 1) / PG::kCommitThreads;
  const cudaError_t e = b2a_host::launch(PG::tree_commit_kernel, dim3(static_cast<unsigned>(gx < 64 ? gx : 64), B),
                                         dim3(PG::kCommitThreads), 0, static_cast<cudaStream_t>(stream), c);
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "tree_commit launch");
}

}  // extern "C"
