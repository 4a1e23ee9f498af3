// Which drafted tokens stand, by sampling (b2a_verify_picks).
//
// At a node of the path the model's next token has weights r = e^((x - M) / T)
// (x its logits row, M the row's largest).  Its children are looked at in order;
// a child with token v and random number u in [0, 1) is accepted if
//   u q(v) < r(v) / sum r
// where q is the row its siblings were drawn from, or 1 where the drafts are
// certain.  A rejected child takes its share out: r(v) = 0 (certain drafts), or
// r = max(r / sum r - q, 0).  Where no child is accepted, the draw d in [0, 1)
// takes the first token v with r(0) + .. + r(v) > d sum r: over all u and d the
// next token then has the model's distribution, whatever was drafted.
//
// Where a residual has no weight left (draft rows that do not sum to 1), the row's
// largest token is taken, and the path goes on to a child that has it.
//
// Only rows on the path decide anything, so only those are read: a cluster of CTAs
// walks one request, each CTA a slice of the vocabulary, and meets over
// distributed shared memory once per row.  The decisions compare sums of 32-bit
// exponentials: up to five multiplied (2^-22 each), arguments of three roundings, 16 or 32
// added in 32 bits (7 roundings deep) and those in 64, so that a sum of weights e^-y is
// off by at most 2^-22 (7 + y) of each; where less than a sixteenth of such a sum is left,
// it is taken anew in 64 bits.  The draw and the residuals, whose outcome hangs on sums at borders some 10^-5
// apart, take 64-bit exponentials: another reading of the row, out of L2.
//
// Bound by latency, not by bytes: a row on a path takes some 7 us (2.5 of loads, 1.5 of
// reductions and the cluster's barrier, 1.5 of the children), a 64-bit sum over it 10 to
// 14 (chains of some 15 dependent operations a token, four side by side).  64 requests
// with up to 31 nodes over 128256 f32 logits: 50 to 73 us, by the longest path, 60 on
// average over eight draws of the inputs; 24 requests with drafts' rows 57 to 75, 65; one
// request of 4 nodes 9 to 19.  With sums in 32 bits throughout 58 us for the 64.  Not kept:
// the next loads or the children's logits ahead of time (registers: 12 % more for the 64),
// more registers and fewer CTAs an SM (half as much again).

#include <cooperative_groups.h>

#include <cfloat>

#include "b2a_common.cuh"

namespace b2a {
namespace verify {

constexpr int kCluster = 8;
constexpr int kMaxNodes = B2A_TREE_MAX_NODES;

struct Args {
  const void* logits;
  long long stride;
  const float* draft;
  long long draft_stride;
  const int *cu, *parents, *tokens;
  const float *uniforms, *draws, *temperature;
  int* picks;
  int B, n_tok, max_nodes, V;
  int all_nodes;  // a cluster per node (verify_path_kernel follows) rather than per request
  int slice, warp_slice, warp_groups;  // tokens of a CTA, of a warp of it, that in groups of 128
};

// e^y in 64 bits (relative error about 10^-13) from y log2(e) x kTable between about -kTable
// x 1000 and 0:  n + f with n whole, a table of 2^(i / kTable) and the series of 2^(f /
// kTable), |f| <= 1/2, up to f^4.
constexpr int kTable = 64;
__device__ __forceinline__ double exp_below(double y, const double* table) {
  constexpr double kRound = 6755399441055744.0;  // 1.5 x 2^52: the sum's low bits are the whole part
  constexpr double c = 0.6931471805599453 / kTable;
  const double t = y + kRound;
  const int n = __double2loint(t);
  const double f = y - (t - kRound);
  double p = fma(f, c * c * c * c / 24.0, c * c * c / 6.0);
  p = fma(f, p, c * c / 2.0);
  p = fma(f, p, c);
  p = fma(f, p, 1.0);
  p *= table[n & (kTable - 1)];
  return __hiloint2double(__double2hiint(p) + (n & ~(kTable - 1)) * ((1 << 20) / kTable), __double2loint(p));
}

struct Exchange {
  double sum, part;  // part: sum of exponentials relative to
  float top;         // the largest logit
  int at;            // the largest's lowest place
};

template <typename T>
__device__ __forceinline__ float at(const T* row, int v) { return ld_elem(row + v); }

// kDraft: drafts have a row.
template <typename T, int kThreads, bool kDraft>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) verify_kernel(const __grid_constant__ Args a) {
  namespace cg = cooperative_groups;
  constexpr int kWarps = kThreads / 32;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) double s_group[];  // sums of the warps' groups of 128 tokens
  uint32_t* gone = reinterpret_cast<uint32_t*>(s_group + kWarps * a.warp_groups);  // bit v of the CTA's
                                                                  // slice: rejected at this node
  __shared__ double s_table[kTable];
  __shared__ Exchange s_ex[2];
  __shared__ double s_warp[kWarps], s_part[kWarps];
  __shared__ float s_top[kWarps];
  __shared__ int s_at[kWarps];
  __shared__ int s_par[kMaxNodes], s_tok[kMaxNodes], s_pick[kMaxNodes];
  __shared__ float s_u[kMaxNodes];
  __shared__ int s_rej[kMaxNodes];      // tokens rejected at this node
  __shared__ double s_mass[kMaxNodes], s_per[kMaxNodes];  // sums of the residuals after each, 1 / them
  pdl_wait();
  const int ranks = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  int b = blockIdx.x / ranks, first = 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (a.all_nodes) {
    // the request of node row b: the last that begins at or before it
    const int node = b;
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu[mid] <= node) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    first = node - a.cu[b];
    // padding, or numbers that are out of bounds (verify_path_kernel records them)
    if (first < 0 || node >= a.cu[b + 1] || a.cu[b + 1] - a.cu[b] > a.max_nodes || a.cu[b] < 0 ||
        a.cu[b + 1] > a.n_tok) {
      if (rank == 0 && tid == 0) a.picks[node] = -1;
      return;  // the whole cluster
    }
  }
  const int c0 = a.cu[b], c1 = a.cu[b + 1], n = c1 - c0;
  const bool bad = n < 0 || n > a.max_nodes || c0 < 0 || c1 > a.n_tok;
  if (rank == 0 && !a.all_nodes) {
    // rows behind the last node, and of a request that is left out, have no pick
    const int last = max(a.cu[a.B], 0);
    for (int i = last + b * kThreads + tid; i < a.n_tok; i += a.B * kThreads) a.picks[i] = -1;
    if (bad) {
      if (tid == 0) set_dev_error(B2A_ERR_POSITION, b);
      for (int i = max(c0, 0) + tid; i < min(c1, a.n_tok); i += kThreads) a.picks[i] = -1;
    }
  }
  if (bad || n == 0) return;  // the whole cluster
  for (int i = tid; i < n; i += kThreads) {
    const int p = a.parents ? a.parents[c0 + i] : i - 1;
    if (rank == 0 && first == 0 && p != -1 && (p < 0 || p >= i)) set_dev_error(B2A_ERR_POSITION, b);
    s_par[i] = p >= 0 && p < i ? p : -1;
    s_tok[i] = a.tokens[c0 + i];
    s_u[i] = a.uniforms[c0 + i];
    s_pick[i] = -1;
  }
  const int v0 = min(rank * a.slice, a.V), v1 = min(v0 + a.slice, a.V);
  for (int i = tid; i < (a.slice + 31) / 32; i += kThreads) gone[i] = 0u;
  if (tid < kTable) s_table[tid] = exp2(tid * (1.0 / kTable));
  __syncthreads();
  const float heat = a.temperature ? (a.temperature[b] > FLT_MAX ? FLT_MAX : a.temperature[b]) : 1.f;
  const bool greedy = !(heat > 0.f);
  const double cold = greedy ? 0.0 : 1.0 / static_cast<double>(heat);
  const double cold_t = cold * 1.4426950408889634 * kTable;
  const float cold2 = static_cast<float>(fmin(cold * 1.4426950408889634, static_cast<double>(FLT_MAX)));
  int buf = 0;

  // what the CTAs of the cluster put into s_ex[buf], combined by all of them alike
  auto exchange_sum = [&](double mine) {
    if (tid == 0) s_ex[buf].sum = mine;
    cluster.sync();
    double sum = lane < ranks ? cluster.map_shared_rank(&s_ex[buf], lane)->sum : 0.0;
#pragma unroll
    for (int o = kCluster / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    buf ^= 1;
    return __shfl_sync(0xffffffffu, sum, 0);
  };

  int cur = first;
  while (true) {
    const T* row = static_cast<const T*>(a.logits) + (c0 + cur) * a.stride;
    const float* qrow = kDraft ? a.draft + (c0 + cur) * a.draft_stride : nullptr;
    // ---- the row's largest logit, its place, the sum of exponentials -----------------
    // (ref: what part is relative to.  It follows top only when that is more than a factor
    // of 2 above it, so that a row that rises in small steps does not round part at each.)
    float top = -INFINITY, ref = -INFINITY;
    double part = 0.0;
    float some = 0.f;  // (of up to kLoads groups, then added to part)
    int place = a.V;
    {
      constexpr int kVec = 16 / sizeof(T), kLoads = 4;
      auto take = [&](const float* x, int v, int apart) {  // kVec logits from v on
        float m = x[0];
#pragma unroll
        for (int e = 1; e < kVec; ++e) m = fmaxf(m, x[e]);
        if (m > top) {
          top = m;
          if ((m - ref) * cold2 > 1.f) {
            const float f = fast_exp2((ref - m) * cold2);
            part *= f;
            some *= f;
            ref = m;
          }
#pragma unroll
          for (int e = kVec - 1; e >= 0; --e)
            if (x[e] == m) place = v + e * apart;
        }
        if (top > -INFINITY) {
          float y[kVec];
#pragma unroll
          for (int e = 0; e < kVec; ++e) y[e] = fast_exp2((x[e] - ref) * cold2);
#pragma unroll
          for (int k = 1; k < kVec; k *= 2)
#pragma unroll
            for (int e = 0; e < kVec; e += 2 * k) y[e] += y[e + k];
          some += y[0];
        }
      };
      if (reinterpret_cast<uintptr_t>(row) % 16 == 0) {  // (slices are whole groups)
        const int groups = (v1 - v0) / kVec;
        for (int i0 = tid; i0 < groups; i0 += kThreads * kLoads) {
          uint4 u[kLoads];
#pragma unroll
          for (int k = 0; k < kLoads; ++k) {
            const int i = i0 + k * kThreads;
            if (i < groups) u[k] = __ldg(reinterpret_cast<const uint4*>(row + v0) + i);
          }
#pragma unroll
          for (int k = 0; k < kLoads; ++k) {
            const int i = i0 + k * kThreads;
            if (i >= groups) continue;
            float x[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e)  // (a NaN has weight 0)
              x[e] = fmaxf(ld_elem(reinterpret_cast<const T*>(&u[k]) + e), -INFINITY);
            take(x, v0 + i * kVec, 1);
          }
          part += some;
          some = 0.f;
        }
        for (int v = v0 + groups * kVec + tid; v < v1; v += kThreads) {
          float x[kVec];
          x[0] = fmaxf(at(row, v), -INFINITY);
#pragma unroll
          for (int e = 1; e < kVec; ++e) x[e] = -INFINITY;
          take(x, v, 1);
        }
        part += some;
      } else {
        for (int v = v0 + tid; v < v1; v += kThreads * kVec) {
          float x[kVec];
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            x[e] = v + e * kThreads < v1 ? fmaxf(at(row, v + e * kThreads), -INFINITY) : -INFINITY;
          take(x, v, kThreads);
          part += some;
          some = 0.f;
        }
      }
    }
    // The lowest place of the largest, the sum relative to it: of a warp's lanes.
    auto join = [&]() {
      const uint32_t u = __float_as_uint(top);  // (in the order of the floats)
      const uint32_t key = (u & 0x80000000u) ? ~u : u | 0x80000000u;
      const uint32_t most = __reduce_max_sync(0xffffffffu, key);
      const float all = __uint_as_float((most & 0x80000000u) ? most ^ 0x80000000u : ~most);
      place = __reduce_min_sync(0xffffffffu, top == all ? place : a.V);
      part = top > -INFINITY ? part * fast_exp2((ref - all) * cold2) : 0.0;
      top = ref = all;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    };
    join();
    if (lane == 0) {
      s_top[warp] = top;
      s_part[warp] = part;
      s_at[warp] = place;
    }
    __syncthreads();
    if (warp == 0) {
      top = ref = lane < kWarps ? s_top[lane] : -INFINITY;
      part = lane < kWarps ? s_part[lane] : 0.0;
      place = lane < kWarps ? s_at[lane] : a.V;
      join();
      if (lane == 0) {
        s_ex[buf].top = top;
        s_ex[buf].part = part;
        s_ex[buf].at = place;
      }
    }
    cluster.sync();
    {
      const Exchange* e = cluster.map_shared_rank(&s_ex[buf], lane < ranks ? lane : 0);
      top = ref = lane < ranks ? e->top : -INFINITY;
      part = lane < ranks ? e->part : 0.0;
      place = lane < ranks ? e->at : a.V;
      join();
    }
    buf ^= 1;
    if (!(top > -INFINITY)) {  // nothing can be picked
      if (rank == 0 && tid == 0) s_pick[cur] = -1;
      place = -1;
    }
    const bool sure = greedy || top == INFINITY || place < 0;  // the largest, or nothing
    const double M = top;
    // ---- the children in order ----------------------------------------------------------
    int rejected = 0, next = -1;
    double total = part;  // sum of r (certain drafts); drafts with a row: r is relative to it
    // e^((x - M) / T).  Weights below e^-690 are 0, and a NaN's; the exponent itself is
    // compared: a float next to M may be off by more where T is small.
    auto weight = [&](float x) {
      constexpr double least = -690.0 * 1.4426950408889634 * kTable;
      const double y = (static_cast<double>(x) - M) * cold_t, e = exp_below(y, s_table);
      return y >= least ? e : 0.0;
    };
    // r(v) after k rejections of drafts with a row, from e^((x - M) / T)
    double per_total = 1.0 / total;
    auto residual = [&](double e, float q, int k) {
      const double p = q;
      double r = fma(e, per_total, -p);
      for (int i = 1; i <= k; ++i) {
        r = r > 0.0 ? r : 0.0;
        if (i < k) r = fma(r, s_per[i - 1], -p);
      }
      return k ? r : e * per_total;
    };
    const bool whole = reinterpret_cast<uintptr_t>(row) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(qrow) % 16 == 0;  // (slices are whole groups)
    // 4 consecutive tokens' logits and draft probabilities; what is left of them after k
    // rejections (the rejected themselves apart).  The tokens go through each step side by
    // side: a chain of 64-bit operations is long.
    auto load4 = [&](int v, int k, float* x, float* q) {
      if (whole && v + 4 <= v1) {
        paged::load4(row + v, x);
        if (kDraft && k) paged::load4(qrow + v, q);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = v + e < v1 ? at(row, v + e) : -INFINITY;
          q[e] = kDraft && k && v + e < v1 ? qrow[v + e] : 0.f;
        }
      }
    };
    auto left4 = [&](int v, int k, const float* x, const float* q, double* r) {
      const uint32_t marks = v < v1 ? gone[(v - v0) >> 5] >> ((v - v0) & 31) : 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = weight(x[e]);
      if (kDraft && k) {
        double per = per_total;
        for (int i = 0; i < k; ++i) {
          if (i) per = s_per[i - 1];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double y = fma(r[e], per, -static_cast<double>(q[e]));
            r[e] = y > 0.0 ? y : 0.0;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = (marks >> e & 1u) ? 0.0 : r[e];
    };
    // The sum of it over the row; those of the warps' groups stay in s_group, the warps'
    // in s_warp, the CTA's in s_ex (the other buffer).
    auto mass = [&](int k) {
      double sum = 0.0;
      const int lo = v0 + warp * a.warp_slice;
      float x[4], q[4], x_next[4], q_next[4];
      load4(lo + 4 * lane, k, x_next, q_next);
      for (int i = 0; i < a.warp_groups && lo + 128 * i < v1; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = x_next[e];
          q[e] = q_next[e];
        }
        if (i + 1 < a.warp_groups) load4(lo + 128 * (i + 1) + 4 * lane, k, x_next, q_next);
        double r[4];
        left4(lo + 128 * i + 4 * lane, k, x, q, r);
        double s = (r[0] + r[1]) + (r[2] + r[3]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) s_group[warp * a.warp_groups + i] = s;
        sum += s;
      }
      __syncthreads();  // (s_warp has been read)
      if (lane == 0) s_warp[warp] = sum;
      __syncthreads();
      double mine = lane < kWarps ? s_warp[lane] : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
      return exchange_sum(mine);
    };
    bool exact = false;  // total is the 64-bit sum of all weights (certain drafts: of those left)
    double left = 0.0;   // what the draw takes from
    int child = cur;
    while (true) {
      int ask = -1;  // rejections behind which a sum is needed before the next child
      while (place >= 0) {
        // the next child
        int c = kMaxNodes;
#pragma unroll
        for (int w = 0; w < kMaxNodes / 32; ++w) {
          const int j = w * 32 + lane;
          const unsigned hit = __ballot_sync(0xffffffffu, j > child && j < n && s_par[j] == cur);
          if (c == kMaxNodes && hit) c = w * 32 + __ffs(hit) - 1;
        }
        if (c == kMaxNodes) break;
        child = c;
        const int v = s_tok[c];
        if (v < 0 || v >= a.V) continue;
        if (sure) {
          if (v == place) {
            next = c;
            break;
          }
          continue;
        }
        bool again = false;
        for (int i = lane; i < rejected; i += 32) again |= s_rej[i] == v;
        again = __any_sync(0xffffffffu, again);
        const double u = s_u[c];
        const double e = weight(at(row, v));
        if constexpr (!kDraft) {
          if (again) continue;
          if (u * total < e) {
            next = c;
            break;
          }
          total -= e;
        } else {
          const float q = __ldg(qrow + v);
          const double r = again ? 0.0 : residual(e, q, rejected);
          if (u * static_cast<double>(q) * (rejected ? s_mass[rejected - 1] : 1.0) < r) {
            next = c;
            break;
          }
        }
        __syncthreads();  // all have read s_rej
        if (tid == 0) {
          s_rej[rejected] = v;
          const int w = v - v0;
          if (v >= v0 && v < v1) gone[w >> 5] |= 1u << (w & 31);
        }
        ++rejected;
        __syncthreads();
        if (kDraft) {
          ask = exact ? rejected : 0;
          break;
        }
        // (where little is left of the 32-bit sum, the rest is summed up by itself)
        if (!exact && total < 0.0625 * part) {
          ask = 0;
          break;
        }
      }
      if (next >= 0 || sure) break;
      if (kDraft && ask < 0 && rejected) {
        left = s_mass[rejected - 1];
        break;
      }
      double sum;
      while (true) {
        sum = mass(max(ask, 0));
        if (!kDraft || ask != 0) break;
        total = sum + weight(at(row, s_rej[0]));  // (the weights' own sum counts the rejected token too)
        per_total = 1.0 / total;
        ask = rejected;
      }
      exact = true;
      if (ask < 0) {
        left = sum;
        break;
      }
      if constexpr (kDraft) {
        if (tid == 0) {
          s_mass[rejected - 1] = sum;
          s_per[rejected - 1] = sum > 0.0 ? 1.0 / sum : 0.0;
        }
        __syncthreads();
      } else {
        total = sum;
      }
    }
    if (next < 0 && !sure && !(left > 0.0)) {
      // the largest is taken, and the path goes on to a child that has it as its token
#pragma unroll
      for (int w = 0; w < kMaxNodes / 32; ++w) {
        const int j = w * 32 + lane;
        const unsigned hit = __ballot_sync(0xffffffffu, j > cur && j < n && s_par[j] == cur && s_tok[j] == place);
        if (next < 0 && hit) next = w * 32 + __ffs(hit) - 1;
      }
    }
    if (next >= 0 && a.all_nodes) {
      if (rank == 0 && tid == 0) a.picks[c0 + cur] = s_tok[next];
      break;
    }
    if (next >= 0) {
      if (rank == 0 && tid == 0) s_pick[cur] = s_tok[next];
      __syncthreads();
      for (int i = tid; i < rejected; i += kThreads) {  // the next row has no marks
        const int w = s_rej[i] - v0;
        if (s_rej[i] >= v0 && s_rej[i] < v1) gone[w >> 5] = 0u;
      }
      __syncthreads();
      cur = next;
      continue;
    }
    // ---- nothing drafted follows: the draw --------------------------------------------
    int drawn = place;  // the largest, -1 for nothing
    if (!sure) {
      const int k = kDraft ? rejected : 0;
      const Exchange* ex = &s_ex[buf ^ 1];
      if (left > 0.0) {
        const double goal = static_cast<double>(a.draws[b]) * left;
        // the CTA and the warp in which the running sum passes the goal
        double before = 0.0;
        int who = -1;
        double who_before = 0.0;
        for (int r = 0; r < ranks; ++r) {
          const double s = cluster.map_shared_rank(ex, r)->sum;
          if (s > 0.0 && (who < 0 || who_before + cluster.map_shared_rank(ex, who)->sum <= goal)) {
            who = r;
            who_before = before;
          }
          before += s;
        }
        drawn = -2;  // another CTA's
        if (who == rank) {
          double wb = who_before, ww_before = 0.0;
          int ww = -1;
          for (int w = 0; w < kWarps; ++w) {
            if (s_warp[w] > 0.0 && (ww < 0 || ww_before + s_warp[ww] <= goal)) {
              ww = w;
              ww_before = wb;
            }
            wb += s_warp[w];
          }
          if (ww == warp) {
            // the group of 128 tokens, then the token; of the last bits that sums
            // in another order differ by, the last token with a weight makes up
            const int lo = v0 + warp * a.warp_slice;
            double run = ww_before, group_before = ww_before;
            int group = 0;
            bool passed = false;
            for (int i = 0; i < a.warp_groups && lo + 128 * i < v1 && !passed; ++i) {
              const double s = s_group[warp * a.warp_groups + i];
              if (s > 0.0) {
                group = i;
                group_before = run;
                passed = run + s > goal;
              }
              run += s;
            }
            const int v = lo + 128 * group + 4 * lane;
            float x[4], q[4];
            double r[4];
            load4(v, k, x, q);
            left4(v, k, x, q, r);
            double inc = (r[0] + r[1]) + (r[2] + r[3]);
            const double mine = inc;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double y = __shfl_up_sync(0xffffffffu, inc, o);
              if (lane >= o) inc += y;
            }
            double cum = group_before + (inc - mine);
            int found = -1, last = -1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              cum += r[e];
              if (r[e] > 0.0) {
                last = v + e;
                if (found < 0 && cum > goal) found = v + e;
              }
            }
            const unsigned pass = __ballot_sync(0xffffffffu, found >= 0);
            const unsigned some = __ballot_sync(0xffffffffu, last >= 0);
            const int pick = pass ? __shfl_sync(0xffffffffu, found, __ffs(pass) - 1)
                                  : __shfl_sync(0xffffffffu, last, some ? 31 - __clz(some) : 0);
            if (lane == 0) a.picks[c0 + cur] = pick;
          }
        }
      }
    }
    if (rank == 0) {
      __syncthreads();
      if (!a.all_nodes)
        for (int i = tid; i < n; i += kThreads)
          if (i != cur) a.picks[c0 + i] = s_pick[i];
      if (tid == 0 && drawn > -2) a.picks[c0 + cur] = drawn;
    }
    break;
  }
  cluster.sync();  // no CTA leaves while others read its shared memory
}

// Behind a cluster per node: the picks of nodes off the path become -1.  The child
// that was accepted is the first whose token is the pick (a token that a sibling
// had is never accepted again, and the draw leaves out the children's tokens).  A warp
// per request.
constexpr int kPathWarps = 4;
__global__ void __launch_bounds__(kPathWarps * 32) verify_path_kernel(const __grid_constant__ Args a) {
  pdl_wait();
  const int b = blockIdx.x * kPathWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (b >= a.B) return;
  const int c0 = a.cu[b], n = a.cu[b + 1] - c0;
  if (n < 0 || n > a.max_nodes || c0 < 0 || c0 + n > a.n_tok) {
    if (lane == 0) set_dev_error(B2A_ERR_POSITION, b);
    return;
  }
  int par[kMaxNodes / 32], tok[kMaxNodes / 32], pick[kMaxNodes / 32];
  bool on[kMaxNodes / 32];
#pragma unroll
  for (int w = 0; w < kMaxNodes / 32; ++w) {
    const int j = w * 32 + lane;
    par[w] = j < n ? (a.parents ? a.parents[c0 + j] : j - 1) : -2;
    tok[w] = j < n ? a.tokens[c0 + j] : -1;
    pick[w] = j < n ? a.picks[c0 + j] : -1;
    on[w] = false;
  }
  int cur = n > 0 ? 0 : -1;
  while (cur >= 0) {
    int want = -1;
#pragma unroll
    for (int w = 0; w < kMaxNodes / 32; ++w) {
      if (w == cur >> 5) want = __shfl_sync(0xffffffffu, pick[w], cur & 31);
      if (w * 32 + lane == cur) on[w] = true;
    }
    int next = -1;
#pragma unroll
    for (int w = 0; w < kMaxNodes / 32; ++w) {
      const unsigned hit = __ballot_sync(0xffffffffu, want >= 0 && par[w] == cur && w * 32 + lane > cur && tok[w] == want);
      if (next < 0 && hit) next = w * 32 + __ffs(hit) - 1;
    }
    cur = next;
  }
#pragma unroll
  for (int w = 0; w < kMaxNodes / 32; ++w)
    if (w * 32 + lane < n && !on[w]) a.picks[c0 + w * 32 + lane] = -1;
}

}  // namespace verify
}  // namespace b2a

// ===========================================================================
// Host side
// ===========================================================================
namespace {

namespace VF = b2a::verify;

template <typename T, int kThreads>
cudaError_t verify_launch(VF::Args a, cudaStream_t st) {
  // whole groups of 128 tokens for each warp
  constexpr int kWarps = kThreads / 32;
  a.warp_groups = (a.V + VF::kCluster * kWarps * 128 - 1) / (VF::kCluster * kWarps * 128);
  a.warp_slice = a.warp_groups * 128;
  a.slice = a.warp_slice * kWarps;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.all_nodes ? a.n_tok : a.B) * VF::kCluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kWarps * a.warp_groups * sizeof(double) + (a.slice + 31) / 32 * 4;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = VF::kCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (b2a_host::launch_flags() & B2A_LAUNCH_PDL) ? 2 : 1;
  // (with what stands in it besides, more than 48 KB from some 1,800,000 tokens on)
  auto* kernel = a.draft ? &VF::verify_kernel<T, kThreads, true> : &VF::verify_kernel<T, kThreads, false>;
  static std::atomic<unsigned long long> done[2];
  cudaError_t e = allow_smem(kernel, 64 * 1024, done[a.draft ? 1 : 0]);
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e == cudaSuccess && a.all_nodes)
    e = launch_second(VF::verify_path_kernel, dim3((a.B + VF::kPathWarps - 1) / VF::kPathWarps),
                      dim3(VF::kPathWarps * 32), 0, st, a);
  return e;
}

}  // namespace

extern "C" {

int b2a_verify_picks(const void* logits, long long row_stride, int dtype, const float* draft,
                     long long draft_row_stride, const int* cu_dev, const int* parents_dev,
                     const int* tokens_dev, const float* uniforms_dev, const float* draws_dev,
                     const float* temperature_dev, int* picks_dev, int B, int n_rows, int max_nodes,
                     int V, void* stream) {
  if (!logits || !cu_dev || !tokens_dev || !uniforms_dev || !draws_dev || !picks_dev)
    return fail(B2A_ERR_ARG, "verify_picks: null pointer argument");
  if (B <= 0 || n_rows < 0 || V <= 0)
    return fail(B2A_ERR_ARG, "verify_picks: sizes must be positive (B=%d n_rows=%d V=%d)", B, n_rows, V);
  if (max_nodes <= 0 || max_nodes > B2A_TREE_MAX_NODES)
    return fail(B2A_ERR_ARG, "verify_picks: max_nodes %d (1..%d)", max_nodes, B2A_TREE_MAX_NODES);
  const int es = b2a_host::elem_size(dtype);
  if (es == 0) return fail(B2A_ERR_DTYPE, "verify_picks: dtype %d", dtype);
  if (row_stride < V || (draft && draft_row_stride < V))
    return fail(B2A_ERR_SHAPE, "verify_picks: row strides %lld, %lld < V=%d", row_stride, draft_row_stride, V);
  if (V > 2000000) return fail(B2A_ERR_UNSUPPORTED, "verify_picks: V %d > 2000000", V);
  if (B > INT_MAX / VF::kCluster || n_rows > INT_MAX / VF::kCluster) return fail(B2A_ERR_UNSUPPORTED, "verify_picks: %d requests", B);
  if (reinterpret_cast<uintptr_t>(logits) % es || reinterpret_cast<uintptr_t>(draft) % 4)
    return fail(B2A_ERR_ALIGN, "verify_picks: rows must be aligned to their elements");
  if (n_rows == 0) return B2A_OK;
  VF::Args a = {logits, row_stride, draft, draft_row_stride, cu_dev, parents_dev, tokens_dev, uniforms_dev,
                draws_dev, temperature_dev, picks_dev, B, n_rows, max_nodes, V, 0, 0, 0, 0};
  // Few rows: a cluster for each, all at once, rather than node after node of a path, as
  // long as all clusters are resident (rows of 128256 f32: 4 nodes of one request 8.6 us
  // against 14.8, 8 of each of 4 24.7 against 29.0; of 8 requests 36.7 against 28.8).
  a.all_nodes = n_rows > B && static_cast<long long>(n_rows) * VF::kCluster <= 2 * b2a_host::sm_count();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* t) {
    using T = typename std::remove_pointer<decltype(t)>::type;
    // Wider CTAs where all clusters are resident with them (2 of 512 threads an SM, 4 of
    // 256): 24 requests with drafts' rows 77 us with 256 threads, 65 with 512, 37 requests
    // of 8 nodes 41 with either, 64 requests 52 and 64.
    const long long ctas = static_cast<long long>(a.all_nodes ? n_rows : B) * VF::kCluster;
    return ctas <= 2 * b2a_host::sm_count() ? verify_launch<T, 512>(a, st) : verify_launch<T, 256>(a, st);
  });
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "verify_picks launch");
}

}  // extern "C"
