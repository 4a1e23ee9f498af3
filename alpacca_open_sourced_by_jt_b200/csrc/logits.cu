// Penalties for repeated tokens, logit biases and grammar masks on the rows of
// the LM head, and each row's greedy pick.
//
// Row r (node t of request b), token v:
//   x = logit + bias_b[v]
//   c = times v was said: in the request's output, and on the node's path
//       (its own token and its ancestors')
//   x = x > 0 ? x / repetition : x * repetition     if c > 0 or v is in the prompt
//   x = x - frequency * c;  x = x - presence        if c > 0
//   x = -inf                                        if the grammar forbids v
// every operation rounded once to f32.  The pick is the lowest v of the
// largest x (-1 where no x is above -inf).
//
// Bound by reading and writing the rows, if the few tokens that need more than
// a copy and a mask are kept out of the way of the others.  A CTA takes one
// slice of the vocabulary of one request; from the history, the biases and the
// drafted tokens it builds, once for several rows, the slice's counts in shared
// memory (integer atomics: the order does not matter) and, for each warp, the
// list of the touched ones among the tokens it streams.  For each row a warp
// evaluates its list first, one token to a lane, into shared memory, then
// streams its part of the row through, 16 tokens a thread, taking the touched
// ones from there, with the next row's loads in flight: no barrier of the CTA in
// the loop.  A node's path is added to the counts before its row and taken off
// after it by the warp that has the drafted token.  Each warp leaves its best
// (value, lowest token) as one ordered 64-bit key and a second small kernel
// takes the rows' maxima.  1023 rows of 128256, f32, with masks: 258 us (4.0 TB/s);
// with the divisions where the tokens stand 267, with one list per CTA and a
// barrier a row 395 (the three in turn on one GPU).

#include "b2a_common.cuh"

namespace b2a {
namespace logits {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kEach = 16;                 // tokens of a thread
constexpr int kSlice = kThreads * kEach;  // tokens of a CTA
constexpr int kMaxNodes = B2A_TREE_MAX_NODES;
constexpr int kWords = kMaxNodes / 32;
constexpr uint32_t kPrompt = 0x80000000u;  // the token is in the prompt
constexpr uint32_t kBias = 0x40000000u;    // the token has a bias
constexpr uint32_t kDraft = 0x20000000u;   // the token is drafted in the request's tree
constexpr uint32_t kCount = 0x1fffffffu;

struct Args {
  const void* in;
  long long in_stride;
  void* out;
  long long out_stride;
  const int *cu, *parents, *tokens;
  const int *hist, *hist_start, *prompt_len;
  const float *repetition, *presence, *frequency;
  const int *bias_start, *bias_ids;
  const float* bias;
  const uint32_t* mask;
  long long mask_stride;
  unsigned long long* best;  // [n_rows][slices * kWarps]
  int* picks;
  int n_hist, n_bias, B, n_rows, max_nodes, V, slices, rows_per_cta;
};

// The rows of request b; false for one that is left out (recorded by the first
// kernel): both kernels ask here, since the second reads what the first wrote.
__device__ __forceinline__ bool request_rows(const Args& a, int b, int& c0, int& n) {
  c0 = a.cu[b];
  const int c1 = a.cu[b + 1];
  n = c1 - c0;
  return c0 >= 0 && c1 >= c0 && c1 <= a.n_rows && n <= a.max_nodes;
}

// A value's place in the order of floats, 0 for what cannot be picked (-inf).
__device__ __forceinline__ uint32_t order_of(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <typename T, int W>
__device__ __forceinline__ void load_w(const T* p, float* x) {
  if constexpr (W == 1) {
    x[0] = ld_elem(p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = ld_elem(h + e);
  }
}

template <typename T, int W>
__device__ __forceinline__ void store_w(T* p, const float* x) {
  if constexpr (W == 1) {
    st_elem(p, x[0]);
  } else if constexpr (sizeof(T) == 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
  } else {
    uint2 u;
    u.x = MmaOp<T>::pack(x[0], x[1]);
    u.y = MmaOp<T>::pack(x[2], x[3]);
    __stcs(reinterpret_cast<uint2*>(p), u);
  }
}

// W = 4: rows whose groups of 4 tokens are aligned; W = 1: any.
template <typename TI, typename TO, int W>
__global__ void __launch_bounds__(kThreads, 3) logits_kernel(const __grid_constant__ Args a) {
  pdl_wait();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) uint32_t lsm[];
  uint32_t* info = lsm;               // [kSlice] flags and counts
  uint32_t* bidx = info + kSlice;     // [kSlice] 1 + bias entry
  float* fixed = reinterpret_cast<float*>(bidx + kSlice);  // [kSlice] touched tokens' values
  uint16_t* lists = reinterpret_cast<uint16_t*>(fixed + kSlice);  // [kWarps][kSlice / kWarps] their places
  __shared__ uint32_t s_anc[kMaxNodes][kWords];
  __shared__ int s_par[kMaxNodes], s_tok[kMaxNodes];
  __shared__ uint32_t s_in[kWarps][kWords];  // the nodes whose token is among the warp's
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // slices in the grid's slowest dimension: the first slices, where frequent
  // tokens are and lists are long, start first
  const int b = blockIdx.x, slice = blockIdx.z;
  int c0, n;
  if (!request_rows(a, b, c0, n)) {
    if (tid == 0) set_dev_error(B2A_ERR_POSITION, b);
    return;
  }
  const int t_lo = blockIdx.y * a.rows_per_cta, t_hi = min(n, t_lo + a.rows_per_cta);
  if (t_lo >= t_hi) return;
  const int v_lo = slice * kSlice, v_hi = min(a.V, v_lo + kSlice);

  // group k of this thread: W tokens from v_lo + k * kPass + tid * W on
  constexpr int kGroups = kEach / W;
  constexpr int kPass = kThreads * W;
  const int len = v_hi - v_lo;
  const TI* in = static_cast<const TI*>(a.in) + (static_cast<size_t>(c0) + t_lo) * a.in_stride + v_lo;
  TO* out = static_cast<TO*>(a.out) + (static_cast<size_t>(c0) + t_lo) * a.out_stride + v_lo;
  const uint32_t* mask =
      a.mask ? a.mask + (static_cast<size_t>(c0) + t_lo) * a.mask_stride + (v_lo >> 5) : nullptr;
  float next[kEach];
  uint32_t next_mask[W == 4 ? kGroups : 1];
  auto fetch = [&](const TI* src, const uint32_t* m) {
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int i = k * kPass + tid * W;
      if (i + W <= len) {
        load_w<TI, W>(src + i, next + k * W);
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) next[k * W + e] = i + e < len ? ld_elem(src + i + e) : -INFINITY;
      }
      if constexpr (W == 4) next_mask[k] = m && i < len ? m[i >> 5] : 0xffffffffu;
    }
  };
  fetch(in, mask);

  for (int i = tid * 4; i < 2 * kSlice; i += kThreads * 4)
    *reinterpret_cast<uint4*>(lsm + i) = make_uint4(0u, 0u, 0u, 0u);
  if (tid < kWarps * kWords) s_in[tid / kWords][tid % kWords] = 0u;
  if (tid < n) {
    s_par[tid] = a.parents ? a.parents[c0 + tid] : tid - 1;
    s_tok[tid] = a.tokens ? a.tokens[c0 + tid] : -1;
  }
  __syncthreads();
  if (a.hist) {
    const int h0 = min(max(a.hist_start[b], 0), a.n_hist);
    const int h1 = min(max(a.hist_start[b + 1], h0), a.n_hist);
    const int p1 = h0 + (a.prompt_len ? min(max(a.prompt_len[b], 0), h1 - h0) : 0);
    // several loads a thread in flight: one at a time, a history of thousands
    // took longer than the rows
    constexpr int kLoads = 8;
    for (int i0 = h0 + tid; i0 < h1; i0 += kLoads * kThreads) {
      int v[kLoads];
#pragma unroll
      for (int k = 0; k < kLoads; ++k)
        v[k] = i0 + k * kThreads < h1 ? a.hist[i0 + k * kThreads] : -1;
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        if (v[k] < v_lo || v[k] >= v_hi) continue;
        if (i0 + k * kThreads < p1) atomicOr(&info[v[k] - v_lo], kPrompt);
        else atomicAdd(&info[v[k] - v_lo], 1u);
      }
    }
  }
  int e0 = 0;
  if (a.bias) {
    e0 = min(max(a.bias_start[b], 0), a.n_bias);
    const int e1 = min(max(a.bias_start[b + 1], e0), a.n_bias);
    for (int e = e0 + tid; e < e1; e += kThreads) {
      const int v = a.bias_ids[e];
      if (v < v_lo || v >= v_hi) continue;
      atomicOr(&info[v - v_lo], kBias);
      atomicMax(&bidx[v - v_lo], static_cast<uint32_t>(e - e0 + 1));  // the last entry of an id counts
    }
  }
  if (tid < n) {
    if (s_tok[tid] >= v_lo && s_tok[tid] < v_hi) {
      atomicOr(&s_in[(s_tok[tid] - v_lo) % kPass / (32 * W)][tid >> 5], 1u << (tid & 31));
      atomicOr(&info[s_tok[tid] - v_lo], kDraft);
    }
    uint32_t m[kWords];
#pragma unroll
    for (int w = 0; w < kWords; ++w) m[w] = 0u;
    int p = tid;
    while (true) {
#pragma unroll
      for (int w = 0; w < kWords; ++w)
        if ((p >> 5) == w) m[w] |= 1u << (p & 31);
      const int up = s_par[p];
      if (up < 0 || up >= p) {
        if (up != -1) set_dev_error(B2A_ERR_POSITION, b);
        break;
      }
      p = up;
    }
#pragma unroll
    for (int w = 0; w < kWords; ++w) s_anc[tid][w] = m[w];
  }
  __syncthreads();
  // this thread's touched tokens (the same for all rows), and the warp's list
  uint16_t* list = lists + warp * (kSlice / kWarps);
  uint32_t hits = 0u;
  int n_list = 0;
#pragma unroll
  for (int k = 0; k < kGroups; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int i = k * kPass + tid * W + e;
      const bool hit = info[i] != 0u;
      const unsigned word = __ballot_sync(0xffffffffu, hit);
      if (hit) {
        hits |= 1u << (k * W + e);
        list[n_list + __popc(word & ((1u << lane) - 1u))] = static_cast<uint16_t>(i);
      }
      n_list += __popc(word);
    }
  __syncwarp();

  const float rep = a.repetition ? a.repetition[b] : 1.f;
  const float pres = a.presence ? a.presence[b] : 0.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f;
  // the list's first round of the next row is loaded one row ahead
  const int mine = lane < n_list ? list[lane] : 0;
  float ahead = lane < n_list ? ld_elem(in + mine) : 0.f;
  unsigned long long* best_out =
      a.best + ((static_cast<size_t>(c0) + t_lo) * a.slices + slice) * kWarps + warp;
  // the counts change by `by` for the path of node t's tokens that are this warp's
  auto count_path = [&](int t, uint32_t by) {
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      if ((s_anc[t][w] & s_in[warp][w]) >> lane & 1u) atomicAdd(&info[s_tok[w * 32 + lane] - v_lo], by);
    __syncwarp();
  };
  const bool drafts = (s_in[warp][0] | s_in[warp][1] | s_in[warp][2] | s_in[warp][3]) != 0u;
  static_assert(kWords == 4, "drafts");
  for (int t = t_lo; t < t_hi; ++t) {
    if (n_list > 0) {
      if (drafts) count_path(t, 1u);
      for (int p = lane; p < n_list; p += 32) {
        const int i = list[p];
        const uint32_t w = info[i], c = w & kCount;
        float y = p == lane ? ahead : ld_elem(in + i);
        if (w & kBias) y = __fadd_rn(y, a.bias[e0 + bidx[i] - 1]);
        if (c != 0u || (w & kPrompt)) y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
        y = __fsub_rn(y, __fmul_rn(freq, static_cast<float>(c)));
        if (c != 0u) y = __fsub_rn(y, pres);
        fixed[i] = y;
      }
      if (t + 1 < t_hi && lane < n_list) ahead = ld_elem(in + a.in_stride + mine);
      __syncwarp();
      if (drafts) count_path(t, 0xffffffffu);  // minus one
    }
    float x[kEach];
    uint32_t allowed = 0u;
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = next[e];
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int i = k * kPass + tid * W;
      uint32_t word;
      if constexpr (W == 4) word = next_mask[k];
      else word = mask && i < len ? mask[i >> 5] : 0xffffffffu;
      allowed |= ((word >> (i & 31)) & ((1u << W) - 1u)) << (k * W);
    }
    if (t + 1 < t_hi) fetch(in + a.in_stride, mask ? mask + a.mask_stride : nullptr);
    if (hits != 0u) {
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        if (((hits >> (k * W)) & ((1u << W) - 1u)) == 0u) continue;
        float f[W];
        load_w<float, W>(fixed + k * kPass + tid * W, f);
#pragma unroll
        for (int e = 0; e < W; ++e)
          if ((hits >> (k * W + e)) & 1u) x[k * W + e] = f[e];
      }
    }
    if (allowed != (kEach == 32 ? 0xffffffffu : (1u << kEach) - 1u)) {
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (!((allowed >> e) & 1u)) x[e] = -INFINITY;
    }
    float top = -INFINITY;  // (fmaxf passes NaN over: it cannot be picked)
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int i = k * kPass + tid * W;
#pragma unroll
      for (int e = 0; e < W; ++e) top = fmaxf(top, x[k * W + e]);
      if (i + W <= len) {
        store_w<TO, W>(out + i, x + k * W);
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (i + e < len) st_elem(out + i + e, x[k * W + e]);
      }
    }
    // the warp's largest value, and the lowest token that has it
    const uint32_t order = order_of(top);
    const uint32_t most = __reduce_max_sync(0xffffffffu, order);
    uint32_t at = 0xffffffffu;
    if (most != 0u && order == most) {
#pragma unroll
      for (int k = kGroups - 1; k >= 0; --k)
#pragma unroll
        for (int e = W - 1; e >= 0; --e)
          if (x[k * W + e] == top) at = v_lo + k * kPass + tid * W + e;
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0)
      *best_out = most ? (static_cast<unsigned long long>(most) << 32) | (0xffffffffu - at) : 0ull;
    __syncwarp();  // the values are read: the next row's list may be evaluated
    in += a.in_stride;
    out += a.out_stride;
    if (mask) mask += a.mask_stride;
    best_out += static_cast<size_t>(a.slices) * kWarps;
  }
}

// One warp per row: the largest key of the row's slices.
__global__ void __launch_bounds__(kThreads) logits_pick_kernel(const __grid_constant__ Args a) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= a.n_rows) return;
  // rows of no request (padding), or of one that is left out, have no pick
  bool mine = false;
  for (int b = lane; b < a.B; b += 32) {
    int c0, n;
    mine |= request_rows(a, b, c0, n) && row >= c0 && row < c0 + n;
  }
  const bool good = __any_sync(0xffffffffu, mine) != 0;
  unsigned long long best = 0ull;
  const int k = a.slices * kWarps;
  if (good)
    for (int i = lane; i < k; i += 32) {
      const unsigned long long x = a.best[static_cast<size_t>(row) * k + i];
      best = x > best ? x : best;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, best, o);
    best = x > best ? x : best;
  }
  if (lane == 0) a.picks[row] = best ? static_cast<int>(0xffffffffu - static_cast<uint32_t>(best)) : -1;
}

}  // namespace logits
}  // namespace b2a

// ===========================================================================
// Host side
// ===========================================================================
namespace {

namespace LG = b2a::logits;

int logits_slices(int V) { return (V + LG::kSlice - 1) / LG::kSlice; }

template <typename TI, typename TO, int W>
cudaError_t logits_launch(const LG::Args& a, int chunks, cudaStream_t st) {
  auto kern = LG::logits_kernel<TI, TO, W>;
  constexpr int smem = LG::kSlice * (4 + 4 + 4 + 2);
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = allow_smem(kern, smem, done);
  if (e != cudaSuccess) return e;
  return b2a_host::launch(kern, dim3(a.B, chunks, a.slices), dim3(LG::kThreads), smem, st, a);
}

}  // namespace

extern "C" {

size_t b2a_constrain_logits_workspace_bytes(int n_rows, int V) {
  if (n_rows <= 0 || V <= 0) return 0;
  return static_cast<size_t>(n_rows) * logits_slices(V) * LG::kWarps * 8;
}

int b2a_constrain_logits(const void* logits, long long row_stride, int in_dtype, void* out,
                         long long out_row_stride, int out_dtype, int* picks_dev,
                         const int* cu_dev, const int* parents_dev, const int* tokens_dev,
                         const int* hist_dev, const int* hist_start_dev, int n_hist,
                         const int* prompt_len_dev, const float* repetition_dev,
                         const float* presence_dev, const float* frequency_dev,
                         const int* bias_start_dev, const int* bias_ids_dev,
                         const float* bias_dev, int n_bias, const unsigned int* mask_dev,
                         long long mask_row_stride, int B, int n_rows, int max_nodes, int V,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (!logits || !out || !picks_dev || !cu_dev)
    return fail(B2A_ERR_ARG, "constrain_logits: null pointer argument");
  if (B <= 0 || n_rows < 0 || V <= 0 || n_hist < 0 || n_bias < 0)
    return fail(B2A_ERR_ARG, "constrain_logits: sizes must be positive (B=%d n_rows=%d V=%d)", B, n_rows, V);
  if (max_nodes <= 0 || max_nodes > B2A_TREE_MAX_NODES)
    return fail(B2A_ERR_ARG, "constrain_logits: max_nodes %d (1..%d)", max_nodes, B2A_TREE_MAX_NODES);
  if (B > 65535) return fail(B2A_ERR_UNSUPPORTED, "constrain_logits: %d requests > 65535", B);
  if (hist_dev && !hist_start_dev) return fail(B2A_ERR_ARG, "constrain_logits: history without hist_start");
  if (bias_dev && (!bias_start_dev || !bias_ids_dev))
    return fail(B2A_ERR_ARG, "constrain_logits: biases without bias_start or bias_ids");
  const int ei = b2a_host::elem_size(in_dtype), eo = b2a_host::elem_size(out_dtype);
  if (ei == 0 || eo == 0) return fail(B2A_ERR_DTYPE, "constrain_logits: dtypes %d, %d", in_dtype, out_dtype);
  if (row_stride < V || out_row_stride < V || (mask_dev && mask_row_stride < (V + 31) / 32))
    return fail(B2A_ERR_SHAPE, "constrain_logits: rows of %d tokens need strides of at least %d (masks %d)",
                V, V, (V + 31) / 32);
  if (logits == out && (ei != eo || row_stride != out_row_stride))
    return fail(B2A_ERR_ARG, "constrain_logits: in place needs one type and stride");
  if (n_rows == 0) return B2A_OK;
  const size_t need = b2a_constrain_logits_workspace_bytes(n_rows, V);
  if (!workspace || workspace_bytes < need)
    return fail(B2A_ERR_WORKSPACE, "constrain_logits: workspace %zu bytes < %zu needed", workspace_bytes, need);
  if (reinterpret_cast<uintptr_t>(workspace) & 7u)
    return fail(B2A_ERR_ALIGN, "constrain_logits: workspace must be 8-byte aligned");
  LG::Args a = {};
  a.in = logits;
  a.in_stride = row_stride;
  a.out = out;
  a.out_stride = out_row_stride;
  a.cu = cu_dev;
  a.parents = parents_dev;
  a.tokens = tokens_dev;
  a.hist = hist_dev;
  a.hist_start = hist_start_dev;
  a.prompt_len = prompt_len_dev;
  a.repetition = repetition_dev;
  a.presence = presence_dev;
  a.frequency = frequency_dev;
  a.bias_start = bias_start_dev;
  a.bias_ids = bias_ids_dev;
  a.bias = bias_dev;
  a.mask = mask_dev;
  a.mask_stride = mask_row_stride;
  a.best = static_cast<unsigned long long*>(workspace);
  a.picks = picks_dev;
  a.n_hist = n_hist;
  a.n_bias = n_bias;
  a.B = B;
  a.n_rows = n_rows;
  a.max_nodes = max_nodes;
  a.V = V;
  a.slices = logits_slices(V);
  a.rows_per_cta = 16;
  const int chunks = (max_nodes + a.rows_per_cta - 1) / a.rows_per_cta;
  // 4 logits per access where every row starts on such a boundary
  auto fits = [](const void* p, long long stride, int es) {
    return (reinterpret_cast<uintptr_t>(p) % (4 * es)) == 0 && stride % 4 == 0;
  };
  const bool vec = fits(logits, row_stride, ei) && fits(out, out_row_stride, eo);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = with_type(in_dtype, [&](auto* ti) {
    return with_type(out_dtype, [&](auto* to) {
      using TI = typename std::remove_pointer<decltype(ti)>::type;
      using TO = typename std::remove_pointer<decltype(to)>::type;
      return vec ? logits_launch<TI, TO, 4>(a, chunks, st) : logits_launch<TI, TO, 1>(a, chunks, st);
    });
  });
  if (e == cudaSuccess)
    e = launch_second(LG::logits_pick_kernel, dim3((n_rows + LG::kWarps - 1) / LG::kWarps),
                      dim3(LG::kThreads), 0, st, a);
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "constrain_logits launch");
}

}  // extern "C"
