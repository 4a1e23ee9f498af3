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
// Only rows on the path decide anything, so only those are read: a cluster of CTAs
// walks one request, each CTA a slice of the vocabulary, and meets over
// distributed shared memory once per row.  The decisions compare sums of 32-bit
// exponentials (2^-22) held in 64 bits; the draw, whose outcome hangs on sums at
// borders some 10^-5 apart, takes 64-bit exponentials: a second reading of the
// last row, out of L2.

#include <cooperative_groups.h>

#include "b2a_common.cuh"

namespace b2a {
namespace verify {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
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
  int slice, warp_slice;  // tokens of a CTA and of a warp of it
};

struct Exchange {
  double sum;
  float top, part;  // largest logit, sum of exponentials relative to it
  int at;           // the largest's lowest place
};

template <typename T>
__device__ __forceinline__ float at(const T* row, int v) { return ld_elem(row + v); }

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const __grid_constant__ Args a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ uint32_t gone[];  // bit v of the CTA's slice: rejected at this node
  __shared__ Exchange s_ex[2];
  __shared__ double s_warp[kWarps];
  __shared__ float s_top[kWarps], s_part[kWarps];
  __shared__ int s_at[kWarps];
  __shared__ int s_par[kMaxNodes], s_tok[kMaxNodes], s_pick[kMaxNodes];
  __shared__ float s_u[kMaxNodes];
  __shared__ int s_rej[kMaxNodes];      // tokens rejected at this node
  __shared__ double s_mass[kMaxNodes];  // sums of the residuals after each
  pdl_wait();
  const int ranks = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank()), b = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c0 = a.cu[b], c1 = a.cu[b + 1], n = c1 - c0;
  const bool bad = n < 0 || n > a.max_nodes || c0 < 0 || c1 > a.n_tok;
  if (rank == 0) {
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
    if (rank == 0 && p != -1 && (p < 0 || p >= i)) set_dev_error(B2A_ERR_POSITION, b);
    s_par[i] = p >= 0 && p < i ? p : -1;
    s_tok[i] = a.tokens[c0 + i];
    s_u[i] = a.uniforms[c0 + i];
    s_pick[i] = -1;
  }
  const int v0 = min(rank * a.slice, a.V), v1 = min(v0 + a.slice, a.V);
  for (int i = tid; i < (a.slice + 31) / 32; i += kThreads) gone[i] = 0u;
  __syncthreads();
  const float heat = a.temperature ? a.temperature[b] : 1.f;
  const bool greedy = !(heat > 0.f);
  const double cold = greedy ? 0.0 : 1.0 / static_cast<double>(heat);
  const float cold2 = static_cast<float>(fmin(cold * 1.4426950408889634, 1e30));
  int buf = 0;

  // what the CTAs of the cluster put into s_ex[buf], combined by all of them alike
  auto exchange_sum = [&](double mine) {
    if (tid == 0) s_ex[buf].sum = mine;
    cluster.sync();
    double sum = 0.0;
    for (int r = 0; r < ranks; ++r) sum += cluster.map_shared_rank(&s_ex[buf], r)->sum;
    buf ^= 1;
    return sum;
  };

  int cur = 0;
  while (true) {
    const T* row = static_cast<const T*>(a.logits) + (c0 + cur) * a.stride;
    const float* qrow = a.draft ? a.draft + (c0 + cur) * a.draft_stride : nullptr;
    // ---- the row's largest logit, its place, the sum of exponentials -----------------
    float top = -INFINITY, part = 0.f;
    int place = a.V;
    {
      constexpr int kVec = 16 / sizeof(T), kLoads = 4;
      auto take = [&](const float* x, int v) {  // kVec logits from v on
        float m = x[0];
#pragma unroll
        for (int e = 1; e < kVec; ++e) m = fmaxf(m, x[e]);
        if (m > top) {
          part *= fast_exp2((top - m) * cold2);
          top = m;
#pragma unroll
          for (int e = kVec - 1; e >= 0; --e)
            if (x[e] == m) place = v + e;
        }
        if (top > -INFINITY) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) part += x[e] > -INFINITY ? fast_exp2((x[e] - top) * cold2) : 0.f;
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
            for (int e = 0; e < kVec; ++e) x[e] = ld_elem(reinterpret_cast<const T*>(&u[k]) + e);
            take(x, v0 + i * kVec);
          }
        }
        for (int v = v0 + groups * kVec + tid; v < v1; v += kThreads) {
          float x[kVec];
          x[0] = at(row, v);
#pragma unroll
          for (int e = 1; e < kVec; ++e) x[e] = -INFINITY;
          take(x, v);
        }
      } else {
        for (int v = v0 + tid; v < v1; v += kThreads * kVec) {
          float x[kVec];
#pragma unroll
          for (int e = 0; e < kVec; ++e) x[e] = v + e * kThreads < v1 ? at(row, v + e * kThreads) : -INFINITY;
          float m = x[0];
#pragma unroll
          for (int e = 1; e < kVec; ++e) m = fmaxf(m, x[e]);
          if (m > top) {
            part *= fast_exp2((top - m) * cold2);
            top = m;
#pragma unroll
            for (int e = kVec - 1; e >= 0; --e)
              if (x[e] == m) place = v + e * kThreads;
          }
          if (top > -INFINITY) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) part += x[e] > -INFINITY ? fast_exp2((x[e] - top) * cold2) : 0.f;
          }
        }
      }
    }
    // the lowest place of the largest, the sum relative to it
    auto join = [&](float t2, float p2, int i2) {
      if (t2 > top) {
        part = p2 + (top > -INFINITY ? part * fast_exp2((top - t2) * cold2) : 0.f);
        top = t2;
        place = i2;
      } else {
        part += t2 > -INFINITY ? p2 * fast_exp2((t2 - top) * cold2) : 0.f;
        if (t2 == top) place = min(place, i2);
      }
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float t2 = __shfl_xor_sync(0xffffffffu, top, o), p2 = __shfl_xor_sync(0xffffffffu, part, o);
      join(t2, p2, __shfl_xor_sync(0xffffffffu, place, o));
    }
    if (lane == 0) {
      s_top[warp] = top;
      s_part[warp] = part;
      s_at[warp] = place;
    }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) join(s_top[w], s_part[w], s_at[w]);
      s_ex[buf].top = top;
      s_ex[buf].part = part;
      s_ex[buf].at = place;
    }
    cluster.sync();
    top = -INFINITY;
    part = 0.f;
    place = a.V;
    for (int r = 0; r < ranks; ++r) {
      const Exchange* e = cluster.map_shared_rank(&s_ex[buf], r);
      join(e->top, e->part, e->at);
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
    auto weight = [&](float x) {  // e^((x - M) / T)
      return x > -INFINITY ? exp((static_cast<double>(x) - M) * cold) : 0.0;
    };
    // r(v) after k rejections of drafts with a row, from e^((x - M) / T)
    auto residual = [&](double e, float q, int k) {
      double r = e / total;
      for (int i = 0; i < k; ++i) r = fmax((i ? r / s_mass[i - 1] : r) - static_cast<double>(q), 0.0);
      return r;
    };
    // Sum over the row of what is left after k rejections (the rejected tokens
    // themselves apart); the warps' shares stay in s_warp, the CTA's in s_ex
    // (the other buffer, until the next exchange but one).
    auto mass = [&](int k) {
      double sum = 0.0;
      const int lo = v0 + warp * a.warp_slice, hi = min(lo + a.warp_slice, v1);
      for (int v = lo + lane; v < hi; v += 128) {
        float x[4], q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int w = v + 32 * e;
          x[e] = w < hi ? at(row, w) : -INFINITY;
          q[e] = k && w < hi ? __ldg(qrow + w) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int w = v + 32 * e - v0;
          if (v + 32 * e >= hi || (gone[w >> 5] >> (w & 31) & 1u)) continue;
          const double y = weight(x[e]);
          sum += k ? residual(y, q[e], k) : y;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncthreads();  // s_warp and the marks of rejected tokens
      if (lane == 0) s_warp[warp] = sum;
      __syncthreads();
      double mine = 0.0;
      for (int w = 0; w < kWarps; ++w) mine += s_warp[w];
      return exchange_sum(mine);
    };
    bool exact = false;  // total is the 64-bit sum of all weights
    int child = cur;
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
      if (!qrow) {
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
      if (qrow) {
        if (!exact) {
          // (the weights' own sum counts the rejected token too)
          const double rest = mass(0);
          double lost = weight(at(row, s_rej[0]));
          total = rest + lost;
          exact = true;
        }
        const double left = mass(rejected);
        if (tid == 0) s_mass[rejected - 1] = left;
        __syncthreads();
      }
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
      const int k = qrow ? rejected : 0;
      const double left = k ? s_mass[k - 1] : mass(0);
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
            const int lo = v0 + warp * a.warp_slice, hi = min(lo + a.warp_slice, v1);
            double run = ww_before;
            int found = -1, last = -1;
            for (int v = lo; v < hi && found < 0; v += 32) {
              const int w = v + lane;
              double r = 0.0;
              if (w < hi && !(gone[(w - v0) >> 5] >> ((w - v0) & 31) & 1u)) {
                r = weight(at(row, w));
                if (k) r = residual(r, __ldg(qrow + w), k);
              }
              double inc = r;
#pragma unroll
              for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
              }
              const unsigned pass = __ballot_sync(0xffffffffu, r > 0.0 && run + inc > goal);
              const unsigned some = __ballot_sync(0xffffffffu, r > 0.0);
              if (some) last = v + 31 - __clz(some);
              if (pass) found = v + __ffs(pass) - 1;
              run += __shfl_sync(0xffffffffu, inc, 31);
            }
            // (the sums above and this one differ in their last bits)
            if (lane == 0) a.picks[c0 + cur] = found >= 0 ? found : last;
          }
        }
      }
    }
    if (rank == 0) {
      __syncthreads();
      for (int i = tid; i < n; i += kThreads)
        if (i != cur) a.picks[c0 + i] = s_pick[i];
      if (tid == 0 && drawn > -2) a.picks[c0 + cur] = drawn;
    }
    break;
  }
  cluster.sync();  // no CTA leaves while others read its shared memory
}

}  // namespace verify
}  // namespace b2a

// ===========================================================================
// Host side
// ===========================================================================
namespace {

namespace VF = b2a::verify;

template <typename T>
cudaError_t verify_launch(const VF::Args& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.B * VF::kCluster);
  cfg.blockDim = dim3(VF::kThreads);
  cfg.dynamicSmemBytes = (a.slice + 31) / 32 * 4;
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
  return cudaLaunchKernelEx(&cfg, VF::verify_kernel<T>, a);
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
  if (B > INT_MAX / VF::kCluster) return fail(B2A_ERR_UNSUPPORTED, "verify_picks: %d requests", B);
  if (reinterpret_cast<uintptr_t>(logits) % es || reinterpret_cast<uintptr_t>(draft) % 4)
    return fail(B2A_ERR_ALIGN, "verify_picks: rows must be aligned to their elements");
  if (n_rows == 0) return B2A_OK;
  VF::Args a = {logits, row_stride, draft, draft_row_stride, cu_dev, parents_dev, tokens_dev, uniforms_dev,
                draws_dev, temperature_dev, picks_dev, B, n_rows, max_nodes, V, 0, 0};
  // whole 32-token groups for each warp
  a.warp_slice = (V + VF::kCluster * VF::kWarps * 32 - 1) / (VF::kCluster * VF::kWarps * 32) * 32;
  a.slice = a.warp_slice * VF::kWarps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* t) {
    return verify_launch<typename std::remove_pointer<decltype(t)>::type>(a, st);
  });
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "verify_picks launch");
}

}  // extern "C"
