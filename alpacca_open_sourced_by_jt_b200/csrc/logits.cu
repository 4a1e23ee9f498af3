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
// Bound by reading and writing the rows.  The tokens that need more than a copy
// and a mask are few, but evaluated where they stand they would hold up their
// whole warp (a division each).  A CTA takes one slice of the vocabulary of one
// request; from the history, the biases and the drafted tokens it builds, once
// for several rows, the slice's counts in shared memory (integer atomics: the
// order does not matter), a bit per token that is touched, and a list of the
// touched tokens.  Each row is then streamed through with mask and maximum of
// the untouched tokens while the next row's loads are in flight, and the list's
// tokens are redone, one to a thread.  A node's path is added to the counts
// before its row's list and taken off after it, where a drafted token falls
// into the slice.  Each warp leaves its best (value, lowest token) as one
// ordered 64-bit key and a second small kernel takes the rows' maxima.

#include "b2a_common.cuh"

namespace b2a {
namespace logits {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
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
  int n_hist, n_bias, B, n_rows, max_nodes, V, slice, slices, rows_per_cta;
};

// A value's place in the order of floats, 0 for what cannot be picked (NaN,
// -inf); ties go to the lowest token.
__device__ __forceinline__ unsigned long long key_of(float x, int v) {
  if (!(x > -INFINITY)) return 0ull;
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<unsigned long long>(o) << 32) | (0xffffffffu - static_cast<uint32_t>(v));
}

template <typename T, int W>
__device__ __forceinline__ void load_w(const T* p, float* x) {
  if constexpr (W == 1) {
    x[0] = ld_elem(p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 f = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
  } else {
    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
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

template <typename TI, typename TO, int W>
__global__ void __launch_bounds__(kThreads, 3) logits_kernel(const __grid_constant__ Args a) {
  pdl_wait();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) uint32_t lsm[];
  uint32_t* info = lsm;               // [slice] flags and counts
  uint32_t* bidx = lsm + a.slice;     // [slice] 1 + bias entry
  uint32_t* touched = bidx + a.slice;  // [slice / 32] a bit per token with info
  uint16_t* list = reinterpret_cast<uint16_t*>(touched + a.slice / 32);  // [slice] those tokens
  __shared__ int s_list;              // how many
  __shared__ uint32_t s_anc[kMaxNodes][kWords];
  __shared__ int s_par[kMaxNodes], s_tok[kMaxNodes];
  __shared__ uint32_t s_in[kWords];   // the request's nodes whose token is in the slice
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.y;
  const int c0 = a.cu[b];
  const int n = a.cu[b + 1] - c0;
  if (n < 0 || n > a.max_nodes || c0 < 0 || c0 + n > a.n_rows) {
    if (tid == 0) set_dev_error(B2A_ERR_POSITION, b);
    return;
  }
  const int t_lo = blockIdx.z * a.rows_per_cta, t_hi = min(n, t_lo + a.rows_per_cta);
  if (t_lo >= t_hi) return;
  const int v_lo = blockIdx.x * a.slice, v_hi = min(a.V, v_lo + a.slice);

  for (int i = tid * 4; i < 2 * a.slice; i += kThreads * 4)
    *reinterpret_cast<uint4*>(lsm + i) = make_uint4(0u, 0u, 0u, 0u);
  if (tid < kWords) s_in[tid] = 0u;
  if (tid == 0) s_list = 0;
  if (tid < n) {
    s_par[tid] = a.parents ? a.parents[c0 + tid] : tid - 1;
    s_tok[tid] = a.tokens ? a.tokens[c0 + tid] : -1;
  }
  __syncthreads();
  if (a.hist) {
    const int h0 = min(max(a.hist_start[b], 0), a.n_hist);
    const int h1 = min(max(a.hist_start[b + 1], h0), a.n_hist);
    const int p1 = h0 + (a.prompt_len ? min(max(a.prompt_len[b], 0), h1 - h0) : 0);
#pragma unroll 4
    for (int i = h0 + tid; i < h1; i += kThreads) {
      const int v = a.hist[i];
      if (v < v_lo || v >= v_hi) continue;
      if (i < p1) atomicOr(&info[v - v_lo], kPrompt);
      else atomicAdd(&info[v - v_lo], 1u);
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
      atomicOr(&s_in[tid >> 5], 1u << (tid & 31));
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
  for (int i = tid; i < a.slice; i += kThreads) {  // whole warps: the slice is a multiple of 32
    const bool hit = info[i] != 0u;
    const unsigned word = __ballot_sync(0xffffffffu, hit);
    int at = 0;
    if (lane == 0) {
      touched[i >> 5] = word;
      if (word) at = atomicAdd(&s_list, __popc(word));
    }
    at = __shfl_sync(0xffffffffu, at, 0);
    if (hit) list[at + __popc(word & ((1u << lane) - 1u))] = static_cast<uint16_t>(i);
  }
  __syncthreads();
  const int n_list = s_list;

  const float rep = a.repetition ? a.repetition[b] : 1.f;
  const float pres = a.presence ? a.presence[b] : 0.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f;
  constexpr int kPass = kThreads * W;     // tokens of one pass of the CTA
  constexpr int kBatch = W == 4 ? 4 : 8;  // passes with their loads in flight
  // a whole slice of one batch: the next row's loads go out before this row's work
  const bool ahead = v_hi - v_lo == kBatch * kPass;
  const TI* in0 = static_cast<const TI*>(a.in) + static_cast<size_t>(c0) * a.in_stride;
  float next[kBatch][W];
  if (ahead) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      load_w<TI, W>(in0 + t_lo * a.in_stride + v_lo + k * kPass + tid * W, next[k]);
  }
  for (int t = t_lo; t < t_hi; ++t) {
    const size_t row = static_cast<size_t>(c0) + t;
    bool path = false;
#pragma unroll
    for (int w = 0; w < kWords; ++w) path |= (s_anc[t][w] & s_in[w]) != 0u;
    const bool on_path = path && tid < n && ((s_anc[t][tid >> 5] & s_in[tid >> 5]) >> (tid & 31)) & 1u;
    const TI* in = static_cast<const TI*>(a.in) + row * a.in_stride;
    TO* out = static_cast<TO*>(a.out) + row * a.out_stride;
    const uint32_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    // a thread's tokens ascend, so only a larger value replaces its best
    float top = -INFINITY;
    int at = 0;
    auto keep = [&](float* x, int i, uint32_t bits) {  // mask, and best of the untouched
      const uint32_t hit = touched[i >> 5] >> (i & 31);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (!((bits >> e) & 1u)) x[e] = -INFINITY;
        if (x[e] > top && !((hit >> e) & 1u)) {
          top = x[e];
          at = v_lo + i + e;
        }
      }
    };
    auto allowed = [&](int v) { return mask ? mask[v >> 5] >> (v & 31) : 0xffffffffu; };
    int i0 = 0;
    for (; v_lo + i0 + kBatch * kPass <= v_hi; i0 += kBatch * kPass) {
      float x[kBatch][W];
      uint32_t bits[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int v0 = v_lo + i0 + k * kPass + tid * W;
        if (ahead) {
#pragma unroll
          for (int e = 0; e < W; ++e) x[k][e] = next[k][e];
        } else {
          load_w<TI, W>(in + v0, x[k]);
        }
        bits[k] = allowed(v0);
      }
      if (ahead && t + 1 < t_hi) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          load_w<TI, W>(in + a.in_stride + v_lo + k * kPass + tid * W, next[k]);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = i0 + k * kPass + tid * W;
        keep(x[k], i, bits[k]);
        store_w<TO, W>(out + v_lo + i, x[k]);
      }
    }
    for (int i = i0 + tid * W; v_lo + i < v_hi; i += kPass) {
      const int v0 = v_lo + i, live = min(W, v_hi - v0);
      float x[W];
#pragma unroll
      for (int e = 0; e < W; ++e) x[e] = e < live ? ld_elem(in + v0 + e) : -INFINITY;
      keep(x, i, allowed(v0));
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (e < live) st_elem(out + v0 + e, x[e]);
    }
    unsigned long long best = key_of(top, at);
    if (n_list > 0) {
      if (path) {
        __syncthreads();  // the row before is done with the counts
        if (on_path) atomicAdd(&info[s_tok[tid] - v_lo], 1u);
      }
      __syncthreads();  // the copies are written: the list's tokens go over them
      for (int p = tid; p < n_list; p += kThreads) {
        const int i = list[p], v = v_lo + i;
        const uint32_t w = info[i], c = w & kCount;
        float x = ld_elem(in + v);  // in place: the copy just written, or -inf where masked
        if (w & kBias) x = __fadd_rn(x, a.bias[e0 + bidx[i] - 1]);
        if (c != 0u || (w & kPrompt)) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(c)));
        if (c != 0u) x = __fsub_rn(x, pres);
        if (!(allowed(v) & 1u)) x = -INFINITY;
        st_elem(out + v, x);
        const unsigned long long k = key_of(x, v);
        best = k > best ? k : best;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
      best = k > best ? k : best;
    }
    if (lane == 0) a.best[(row * a.slices + blockIdx.x) * kWarps + warp] = best;
    if (path) {
      __syncthreads();
      if (on_path) atomicSub(&info[s_tok[tid] - v_lo], 1u);
    }
  }
}

// One warp per row: the largest key of the row's slices.
__global__ void __launch_bounds__(kThreads) logits_pick_kernel(const __grid_constant__ Args a) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= a.n_rows) return;
  // rows of no request (padding), or of one with too many nodes, have no pick
  int before = 0;
  for (int b = lane; b < a.B; b += 32) before += a.cu[b + 1] <= row ? 1 : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  const bool good = before < a.B && a.cu[before] <= row && a.cu[before + 1] - a.cu[before] <= a.max_nodes;
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

int logits_slice(int V) {
  int s = 4096;
  while (s > 1024 && s / 2 >= V) s /= 2;
  return s;
}

template <typename TI, typename TO>
cudaError_t logits_launch(const LG::Args& a, int chunks, bool vec, cudaStream_t st) {
  const dim3 grid(a.slices, a.B, chunks);
  const size_t smem = static_cast<size_t>(a.slice) * (4 + 4 + 2) + a.slice / 8;
  if (vec) return b2a_host::launch(LG::logits_kernel<TI, TO, 4>, grid, dim3(LG::kThreads), smem, st, a);
  return b2a_host::launch(LG::logits_kernel<TI, TO, 1>, grid, dim3(LG::kThreads), smem, st, a);
}

}  // namespace

extern "C" {

size_t b2a_constrain_logits_workspace_bytes(int n_rows, int V) {
  if (n_rows <= 0 || V <= 0) return 0;
  const int s = logits_slice(V);
  return static_cast<size_t>(n_rows) * ((V + s - 1) / s) * LG::kWarps * 8;
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
  a.slice = logits_slice(V);
  a.slices = (V + a.slice - 1) / a.slice;
  a.rows_per_cta = 8;
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
      return logits_launch<TI, TO>(a, chunks, vec, st);
    });
  });
  if (e == cudaSuccess)
    e = launch_second(LG::logits_pick_kernel, dim3((n_rows + LG::kWarps - 1) / LG::kWarps),
                      dim3(LG::kThreads), 0, st, a);
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "constrain_logits launch");
}

}  // extern "C"
