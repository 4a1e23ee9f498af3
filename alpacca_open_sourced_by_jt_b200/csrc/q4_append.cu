// RMSNorm of the heads of q and k, RoPE and append into a paged cache in one
// pass (b2a_norm_rope_append_paged, b2a_rope_append_q4), rows of a 4-bit pool
// read back (b2a_q4_rows) and the commit of a draft tree in it
// (b2a_tree_commit_q4).
//
// Per head of q and k:  y = x * s * w,  s = 1 / sqrt(sum x^2 / D + eps), then the
// rotation.  The sum is taken in 64 bits and rounded once, with eps, to 32: the
// factor then does not depend on the order of the sum, nor do the codes of
// values next to a border.  Products and sums are rounded one by one, as
// paged.cu does.
//
// Bound by reading the projections and writing q and the pool, and nearly as much by the
// latency of its instructions (55 % of the issue slots used, L1's data path 60 %).  A thread takes eight pairs of a head, which it rotates
// by itself: 16 consecutive dims, or for neox rows 8 and the 8 that are half the rotation
// further on, so two words of codes; D / 16 lanes a head (with 8 dims a thread the sum, the
// root and the addresses of a head weigh twice as much).  It keeps its head over the tokens,
// so that addresses and roles are found once: 8191 tokens, 32/8 heads x 128, bf16: 53 us
// (3.8 TB/s), 72 with the heads in the inner loop; into 4 bits, 64 wide, and read back 36
// us (6 of them the reading back), 56.  Not kept: rows, cosines and sines through rings in shared memory (51 and 42 us).

#include <cfloat>

#include "q4.cuh"

namespace b2a {
namespace q4 {

struct AppendArgs {
  const void *q, *k, *v;
  long long q_stride, k_stride, v_stride;
  const float *bq, *bk, *bv, *wq, *wk, *cos_tab, *sin_tab;
  const int *pos, *slots;
  void *k_pool, *v_pool, *q_out;  // k_pool: the 4-bit pool, or K rows (and v_pool V rows)
  long long page_stride;          // elements; 4-bit pools: bytes
  long long n_slots;
  double inv_d;  // 1 / D (a power of two: the product is the quotient)
  float eps;
  int tab_rows, page_shift, H, KV, D, n_rot, neox, n_tok;
};

// What a block stands for: the scale of 32 values whose largest (by magnitude;
// the negative one of two) has key, as value_key gives it.
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u << 1 | u >> 31;
}
__device__ __forceinline__ __half block_scale(uint32_t key) {
  if ((key >> 1) > 0x7f800000u) return __ushort_as_half(0x7fff);  // NaN
  const float m = __uint_as_float(key >> 1 | key << 31);
  // 8 significant bits; values above 8 x 8160 saturate, so that d * (code - 8)
  // stays inside f16
  const float d = __bfloat162float(__float2bfloat16_rn(m * -0.125f));
  const uint16_t h = __half_as_ushort(__float2half_rn(fminf(fmaxf(d, -8160.f), 8160.f)));
  return __ushort_as_half((h & 0x7fff) ? h : 0);
}
// The codes of 8 consecutive dims, a word:  floor(x / d + 8.5), the quotient rounded to
// nearest.  It is corrected once from x times the rounded reciprocal (P. Markstein, IBM J.
// Res. Dev. 34, 1990): q + (x - q d) / d with an exact remainder, off by 2^-47 of itself
// before its rounding.  No quotient lies as near to a border of the rounding: with the 8
// significant bits of d, a border times d differs from x by 2^-33 of it at least (equal they
// cannot be: the product of an odd number of 25 bits has more than the 24 of x).
__device__ __forceinline__ uint32_t codes8(const float* x, float d) {
  const float r = __frcp_rn(d);
  const bool far = fabsf(d) == 8160.f;  // (saturated: an infinity has no remainder)
  const float2 r2 = make_float2(r, r), nd = make_float2(-d, -d);
  uint32_t w = 0;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    float2 y = make_float2(x[2 * n], x[2 * n + 1]);
    if (far) y = make_float2(fminf(fmaxf(y.x, -FLT_MAX), FLT_MAX), fminf(fmaxf(y.y, -FLT_MAX), FLT_MAX));
    const float2 q = mul2(y, r2);
    const float2 t = fma2(fma2(fma2(q, nd, y), r2, q), make_float2(1.f, 1.f), make_float2(8.5f, 8.5f));
    // 2^23 + the whole part: its low bits
    w += __float_as_uint(__fadd_rd(fminf(fmaxf(t.x, 0.f), 15.f), 8388608.f)) << (4 * n);
    w += __float_as_uint(__fadd_rd(fminf(fmaxf(t.y, 0.f), 15.f), 8388608.f)) << (4 * n + 16);
  }
  return d == 0.f ? 0x88888888u : w - (0x4b000000u + (0x4b000000u << 4));
}
__device__ __forceinline__ uint32_t largest8(const float* x) {
  uint32_t k = 0;
#pragma unroll
  for (int n = 0; n < 8; ++n) k = max(k, value_key(x[n]));
  return k;
}

constexpr int kThreads = 256;
// Most threads, CTAs per SM of norm_append_kernel: 80 registers each (with 64 the rows on
// their way are spilled).
constexpr int kAppendThreads = 384, kResident = 2;

// 8 elements as loaded.
template <typename TS>
struct Raw {
  uint4 w[sizeof(TS) / 2];
  __device__ __forceinline__ void load(const TS* p) {
    w[0] = reinterpret_cast<const uint4*>(p)[0];
    if constexpr (sizeof(TS) == 4) w[1] = reinterpret_cast<const uint4*>(p)[1];
  }
  __device__ __forceinline__ void floats(float* x) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = ld_elem(reinterpret_cast<const TS*>(w) + e);
  }
};

// Q4: the 4-bit pool; otherwise pools of TK.  A thread keeps its head and goes over tokens;
// while it works on a row the next one comes.
template <typename TS, typename TK, typename TQ, bool Q4, bool kNeox>
__global__ void __launch_bounds__(kAppendThreads, kResident) norm_append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_wait();
  const int D = a.D, L = D >> 4;  // a head's dims and lanes: 4, 8 or 16
  const int u = threadIdx.x & (L - 1);
  const int half = a.n_rot >> 1, all = a.H + 2 * a.KV, step = gridDim.y * blockDim.x / L;
  int h = (blockIdx.y * blockDim.x + threadIdx.x) / L;
  // (the same for all lanes: a warp's lanes leave the loop over heads together)
  for (int wh = (blockIdx.y * blockDim.x + (threadIdx.x & ~31u)) / L; wh < all; wh += step, h += step) {
    const bool none = h >= all, is_q = h < a.H, is_v = h >= a.H + a.KV;
    const int hh = is_q ? h : (is_v ? h - a.H - a.KV : h - a.H);
    // the thread's dims: 8 from lo on and 8 from hi on; its pairs rotate
    const bool turned = 16 * u < a.n_rot && !is_v, split = kNeox && turned;
    const int lo = split ? 8 * u : 16 * u, hi = split ? half + 8 * u : 16 * u + 8;
    const TS* src = static_cast<const TS*>(is_q ? a.q : (is_v ? a.v : a.k)) + hh * D;
    const long long stride = is_q ? a.q_stride : (is_v ? a.v_stride : a.k_stride);
    const float* bias = none ? nullptr : (is_q ? a.bq : (is_v ? a.bv : a.bk));
    const float* w = none || is_v ? nullptr : (is_q ? a.wq : a.wk);
    const bool normed = __any_sync(0xffffffffu, w != nullptr);
    Raw<TS> raw[2];
    float c[8], s[8];
    int p = -1, now = -1;
    auto fetch = [&](int i) {
      if (none) return;
      raw[0].load(src + i * stride + lo);
      raw[1].load(src + i * stride + hi);
    };
    auto fetch_turn = [&]() {  // of the token at p
      if (turned && p >= 0 && p < a.tab_rows) {
        const size_t row = static_cast<size_t>(p) * half + 8 * u;
        paged::load8(a.cos_tab + row, c);
        paged::load8(a.sin_tab + row, s);
      }
    };
    if (static_cast<int>(blockIdx.x) < a.n_tok) {
      fetch(blockIdx.x);
      p = a.pos[blockIdx.x];
      now = a.slots[blockIdx.x];
      fetch_turn();
    }
    for (int i = blockIdx.x; i < a.n_tok; i += gridDim.x) {
      const int next = i + gridDim.x;
      const bool ok = p >= 0 && p < a.tab_rows && now < a.n_slots;
      if (!ok && h == 0 && u == 0) set_dev_error(B2A_ERR_POSITION, i);
      const int slot = now;
      float x[16];
      raw[0].floats(x);
      raw[1].floats(x + 8);
      if (next < a.n_tok) {
        fetch(next);
        p = a.pos[next];
        now = a.slots[next];
      }
      if (!ok) {
        fetch_turn();
        continue;
      }
      if (bias) {
        float b[16];
        paged::load8(bias + hh * D + lo, b);
        paged::load8(bias + hh * D + hi, b + 8);
#pragma unroll
        for (int d = 0; d < 16; ++d) x[d] = __fadd_rn(x[d], b[d]);
      }
      if (normed) {
        double s0 = 0.0, s1 = 0.0;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          s0 = fma(static_cast<double>(x[d]), static_cast<double>(x[d]), s0);
          s1 = fma(static_cast<double>(x[d + 8]), static_cast<double>(x[d + 8]), s1);
        }
        s0 += s1;
        s0 += __shfl_xor_sync(0xffffffffu, s0, 1);
        s0 += __shfl_xor_sync(0xffffffffu, s0, 2);
        if (L > 4) s0 += __shfl_xor_sync(0xffffffffu, s0, 4);
        if (L > 8) s0 += __shfl_xor_sync(0xffffffffu, s0, 8);
        const float f = __frcp_rn(__fsqrt_rn(static_cast<float>(s0 * a.inv_d + static_cast<double>(a.eps))));
        if (w != nullptr) {
          const float2 f2 = make_float2(f, f);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            float g[8];
            paged::load8(w + (part ? hi : lo), g);
#pragma unroll
            for (int n = 0; n < 8; n += 2) {
              float* y = x + 8 * part + n;
              const float2 z = mul2(mul2(make_float2(y[0], y[1]), f2), make_float2(g[n], g[n + 1]));
              y[0] = z.x;
              y[1] = z.y;
            }
          }
        }
      }
      if (turned) {
        if constexpr (kNeox) {
#pragma unroll
          for (int n = 0; n < 8; n += 2) {
            const float2 x0 = make_float2(x[n], x[n + 1]), x1 = make_float2(x[n + 8], x[n + 9]);
            const float2 c2 = make_float2(c[n], c[n + 1]), s2 = make_float2(s[n], s[n + 1]);
            const float2 p0 = mul2(x0, c2), p1 = mul2(x1, s2), p2 = mul2(x0, s2), p3 = mul2(x1, c2);
            x[n] = __fsub_rn(p0.x, p1.x);
            x[n + 1] = __fsub_rn(p0.y, p1.y);
            x[n + 8] = __fadd_rn(p2.x, p3.x);
            x[n + 9] = __fadd_rn(p2.y, p3.y);
          }
        } else {
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const float2 p = mul2(make_float2(x[2 * n], x[2 * n + 1]), make_float2(c[n], c[n]));
            const float2 r = mul2(make_float2(x[2 * n + 1], x[2 * n]), make_float2(s[n], s[n]));
            x[2 * n] = __fsub_rn(p.x, r.x);
            x[2 * n + 1] = __fadd_rn(r.y, p.y);
          }
        }
      }
      fetch_turn();
      if (is_q) {
        TQ* to = static_cast<TQ*>(a.q_out) + (static_cast<size_t>(i) * a.H + h) * D;
        paged::store8(to + lo, x);
        paged::store8(to + hi, x + 8);
      }
      if (slot < 0) continue;
      const long long page = (slot >> a.page_shift) * a.page_stride;
      const int in_page = slot & ((1 << a.page_shift) - 1);
      if constexpr (Q4) {
        if (__all_sync(0xffffffffu, is_q || none)) continue;
        // the largest of the block: 2 lanes hold 16 consecutive dims each; split, 4 lanes
        // hold 8 each of two blocks
        uint32_t ka = largest8(x), kb = largest8(x + 8);
        if (!split) ka = kb = max(ka, kb);
        ka = max(ka, __shfl_xor_sync(0xffffffffu, ka, 1));
        kb = max(kb, __shfl_xor_sync(0xffffffffu, kb, 1));
        const uint32_t oa = __shfl_xor_sync(0xffffffffu, ka, 2), ob = __shfl_xor_sync(0xffffffffu, kb, 2);
        if (split) {
          ka = max(ka, oa);
          kb = max(kb, ob);
        }
        if (is_q || none) continue;
        const __half da = block_scale(ka), db = block_scale(kb);
        unsigned char* g = static_cast<unsigned char*>(a.k_pool) + page +
                           (static_cast<long long>(hh) * ((1 << a.page_shift) >> 4) + (in_page >> 4)) * granule_bytes(D);
        const int r = in_page & 15, ua = lo >> 3, ub = hi >> 3;
        *reinterpret_cast<uint32_t*>(g + (is_v ? v_word(D, r, ua) : k_word(D, r, ua))) = codes8(x, __half2float(da));
        *reinterpret_cast<uint32_t*>(g + (is_v ? v_word(D, r, ub) : k_word(D, r, ub))) = codes8(x + 8, __half2float(db));
        // (the lane with a block's first word writes its scale)
        if ((ua & 3) == 0)
          *reinterpret_cast<__half*>(g + (is_v ? v_scale(D, r, ua >> 2) : k_scale(D, r, ua >> 2))) = da;
        if ((ub & 3) == 0)
          *reinterpret_cast<__half*>(g + (is_v ? v_scale(D, r, ub >> 2) : k_scale(D, r, ub >> 2))) = db;
      } else {
        if (is_q || none) continue;
        TK* row = static_cast<TK*>(is_v ? a.v_pool : a.k_pool) + page +
                  (static_cast<long long>(in_page) * a.KV + hh) * D;
        paged::store8(row + lo, x);
        paged::store8(row + hi, x + 8);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Rows of a 4-bit pool, as values
// ---------------------------------------------------------------------------
// A warp takes a block of 32 dims of one head of 8 tokens, a word a lane: 8 rows side by
// side fill the sectors of V words, 4 words those of K words and of the outputs.
template <typename T>
__global__ void __launch_bounds__(kThreads) q4_rows_kernel(const Pool pool, const int* __restrict__ slots,
                                                           T* __restrict__ k, T* __restrict__ v,
                                                           int n_tok, int KV, int D) {
  pdl_wait();
  const long long n_slots = static_cast<long long>(pool.n_pages) << pool.page_shift;
  const int lane = threadIdx.x & 31, blocks = D >> 5;
  for (long long tok = blockIdx.x * 8LL + (lane >> 2); tok - (lane >> 2) < n_tok; tok += gridDim.x * 8LL) {
    if (tok >= n_tok) continue;
    const int slot = slots[tok];
    if (slot >= n_slots && threadIdx.x < 32 && (lane & 3) == 0) set_dev_error(B2A_ERR_POSITION, static_cast<int>(tok));
    const bool held = slot >= 0 && slot < n_slots;
    const int in_page = slot & ((1 << pool.page_shift) - 1), r = in_page & 15;
    for (int j = threadIdx.x >> 5; j < KV * blocks; j += kThreads / 32) {
      const int h = j / blocks, b = j - h * blocks, u = 4 * b + (lane & 3);
      float x[8], y[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) x[d] = y[d] = 0.f;
      if (held) {
        const unsigned char* g = granule(pool, D, slot >> pool.page_shift, h, in_page);
        const uint32_t kw = *reinterpret_cast<const uint32_t*>(g + k_word(D, r, u));
        const uint32_t vw = *reinterpret_cast<const uint32_t*>(g + v_word(D, r, u));
        const float dk = __half2float(*reinterpret_cast<const __half*>(g + k_scale(D, r, b)));
        const float dv = __half2float(*reinterpret_cast<const __half*>(g + v_scale(D, r, b)));
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const int sh = (d >> 1) * 4 + (d & 1) * 16;
          // (2^23 + code less 2^23 + 8)
          x[d] = dk * (__uint_as_float(0x4b000000u | (kw >> sh & 15u)) - 8388616.f);
          y[d] = dv * (__uint_as_float(0x4b000000u | (vw >> sh & 15u)) - 8388616.f);
        }
      }
      const size_t at = (static_cast<size_t>(tok) * KV + h) * D + 8 * u;
      paged::store8(k + at, x);
      paged::store8(v + at, y);
    }
  }
}

// ---------------------------------------------------------------------------
// The accepted path's rows moved into place (paged.cu has the path)
// ---------------------------------------------------------------------------
// A thread moves one word of K and V of a head of a layer for all rows of the
// path, in path order, and the scales of a block; no row is overwritten before it
// was read, since the row at depth d comes from node path[d] >= d.
__global__ void __launch_bounds__(paged::kCommitThreads) tree_commit_q4_kernel(
    const __grid_constant__ paged::Commit c, const __grid_constant__ Pool pool, int KV, int D) {
  pdl_wait();
  __shared__ int s_path[paged::kMaxNodes];
  __shared__ long long s_from[paged::kMaxNodes], s_to[paged::kMaxNodes];  // page, row in it
  __shared__ int s_n;
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    int len = 0;
    const int m = paged::accepted_path(c, b, s_path, len);
    for (int d = lane; d < m; d += 32) {
      const int from = len + s_path[d], to = len + d;
      long long src = -1, dst = -1;
      if (from != to) {
        if (c.page_shift < 0) {
          src = static_cast<long long>(b) << 32 | from;
          dst = static_cast<long long>(b) << 32 | to;
        } else {
          const int pf = c.table[b * c.table_stride + (from >> c.page_shift)];
          const int pt = c.table[b * c.table_stride + (to >> c.page_shift)];
          const int mask = (1 << c.page_shift) - 1;
          if (pf < 0 || pf >= c.n_pages || pt < 0 || pt >= c.n_pages) {
            set_dev_error(B2A_ERR_POSITION, b);
          } else {
            src = static_cast<long long>(pf) << 32 | (from & mask);
            dst = static_cast<long long>(pt) << 32 | (to & mask);
          }
        }
      }
      s_from[d] = src;
      s_to[d] = dst;
    }
    if (lane == 0) s_n = m;
  }
  __syncthreads();
  const int m = s_n, words = D / 8;
  const long long cols = static_cast<long long>(c.n_layers) * KV * words;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < cols;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int u = static_cast<int>(i % words);
    const long long lh = i / words;
    const int h = static_cast<int>(lh % KV);
    const long long layer = lh / KV * c.layer_bytes;
    for (int d = 0; d < m; ++d) {
      if (s_from[d] < 0) continue;
      const int rf = static_cast<int>(s_from[d] & 0x7fffffff), rt = static_cast<int>(s_to[d] & 0x7fffffff);
      const unsigned char* f = granule(pool, D, s_from[d] >> 32, h, rf) + layer;
      unsigned char* t = granule(pool, D, s_to[d] >> 32, h, rt) + layer;
      const int a = rf & 15, z = rt & 15;
      *reinterpret_cast<uint32_t*>(t + k_word(D, z, u)) = *reinterpret_cast<const uint32_t*>(f + k_word(D, a, u));
      *reinterpret_cast<uint32_t*>(t + v_word(D, z, u)) = *reinterpret_cast<const uint32_t*>(f + v_word(D, a, u));
      if (u < D / 32) {
        *reinterpret_cast<uint16_t*>(t + k_scale(D, z, u)) = *reinterpret_cast<const uint16_t*>(f + k_scale(D, a, u));
        *reinterpret_cast<uint16_t*>(t + v_scale(D, z, u)) = *reinterpret_cast<const uint16_t*>(f + v_scale(D, a, u));
      }
    }
  }
}

}  // namespace q4
}  // namespace b2a

// ===========================================================================
// Host side
// ===========================================================================
namespace {

namespace Q4 = b2a::q4;

// What b2a_norm_rope_append_paged and b2a_rope_append_q4 ask of their common
// arguments.
int norm_append_check(const char* who, const Q4::AppendArgs& a, int in_dtype, int q_out_dtype,
                      int n_pages, int page_rows, int style) {
  if (!a.q || !a.k || !a.v || !a.cos_tab || !a.sin_tab || !a.pos || !a.slots || !a.k_pool || !a.v_pool ||
      !a.q_out)
    return fail(B2A_ERR_ARG, "%s: null pointer argument", who);
  if (a.n_tok < 0 || a.H <= 0 || a.KV <= 0 || a.tab_rows <= 0 || n_pages <= 0)
    return fail(B2A_ERR_ARG, "%s: sizes must be positive (n_tok=%d H=%d KV=%d)", who, a.n_tok, a.H, a.KV);
  if (a.D != 64 && a.D != 128 && a.D != 256)
    return fail(B2A_ERR_UNSUPPORTED, "%s: head_dim %d (64/128/256)", who, a.D);
  if (style != B2A_ROPE_NORM && style != B2A_ROPE_NEOX) return fail(B2A_ERR_ARG, "%s: style %d", who, style);
  if (a.n_rot < 0 || a.n_rot > a.D || a.n_rot % 16 != 0)
    return fail(B2A_ERR_SHAPE, "%s: n_rot %d (a multiple of 16, at most D=%d)", who, a.n_rot, a.D);
  const int es = b2a_host::elem_size(in_dtype), qs = b2a_host::elem_size(q_out_dtype);
  if (es == 0 || qs == 0) return fail(B2A_ERR_DTYPE, "%s: dtypes %d, %d", who, in_dtype, q_out_dtype);
  if (!power_of_two(page_rows))
    return fail(B2A_ERR_SHAPE, "%s: page_rows %d is not a power of two", who, page_rows);
  if ((a.wq || a.wk) && !(a.eps >= 0.f && isfinite(a.eps)))
    return fail(B2A_ERR_ARG, "%s: eps must not be negative", who);
  if (a.q_stride < static_cast<long long>(a.H) * a.D || a.k_stride < static_cast<long long>(a.KV) * a.D ||
      a.v_stride < static_cast<long long>(a.KV) * a.D)
    return fail(B2A_ERR_SHAPE, "%s: token strides overlap the rows", who);
  const void* ptrs[] = {a.q, a.k, a.v, a.q_out, a.k_pool, a.v_pool, a.cos_tab, a.sin_tab, a.bq, a.bk, a.bv, a.wq, a.wk};
  bool ok = (a.q_stride * es) % 16 == 0 && (a.k_stride * es) % 16 == 0 && (a.v_stride * es) % 16 == 0;
  for (const void* p : ptrs) ok = ok && b2a_host::aligned16(p);
  if (!ok) return fail(B2A_ERR_ALIGN, "%s: rows, tables, weights and pools must be 16-byte aligned", who);
  return B2A_OK;
}

template <typename TS, typename TK, typename TQ, bool kQ4>
cudaError_t norm_append_launch(const Q4::AppendArgs& a, cudaStream_t st) {
  // A CTA per token, its threads dealt evenly to rounds over the heads; few tokens: a
  // token's rounds over more CTAs, until there are a few per SM.
  const int all = a.H + 2 * a.KV, lanes = a.D / 16;
  int rounds = (all * lanes + Q4::kAppendThreads - 1) / Q4::kAppendThreads;
  const int threads = ((all + rounds - 1) / rounds * lanes + 31) / 32 * 32;
  const int at_once = threads / lanes;
  rounds = (all + at_once - 1) / at_once;
  const int resident = Q4::kResident * (Q4::kAppendThreads / threads) * b2a_host::sm_count();
  const int enough = (resident + a.n_tok - 1) / a.n_tok;
  const dim3 grid(a.n_tok < resident ? a.n_tok : resident, rounds < enough ? rounds : enough), block(threads);
  if (a.neox) return b2a_host::launch(Q4::norm_append_kernel<TS, TK, TQ, kQ4, true>, grid, block, 0, st, a);
  return b2a_host::launch(Q4::norm_append_kernel<TS, TK, TQ, kQ4, false>, grid, block, 0, st, a);
}

// A 4-bit pool's checks and its description.
int q4_pool_check(const char* who, const void* pool, int n_pages, int page_rows, long long& page_bytes,
                  int KV, int D, bool paged_cache) {
  if (!pool) return fail(B2A_ERR_ARG, "%s: null pointer argument", who);
  if (n_pages <= 0 || page_rows <= 0 || KV <= 0)
    return fail(B2A_ERR_ARG, "%s: sizes must be positive (n_pages=%d page_rows=%d KV=%d)", who, n_pages, page_rows, KV);
  if (D != 64 && D != 128 && D != 256)
    return fail(B2A_ERR_UNSUPPORTED, "%s: head_dim %d (64/128/256)", who, D);
  if (page_rows % 16 != 0 || (paged_cache && !power_of_two(page_rows)))
    return fail(B2A_ERR_SHAPE, "%s: page_rows %d must be a %s from 16 up", who, page_rows,
                paged_cache ? "power of two" : "multiple of 16");
  const long long dense = static_cast<long long>(KV) * (page_rows / 16) * Q4::granule_bytes(D);
  if (dense > INT_MAX) return fail(B2A_ERR_UNSUPPORTED, "%s: pages of %lld bytes", who, dense);
  if (page_bytes == 0) page_bytes = dense;
  if (page_bytes < dense)
    return fail(B2A_ERR_SHAPE, "%s: page_bytes %lld < %lld", who, page_bytes, dense);
  if (!b2a_host::aligned16(pool) || page_bytes % 16 != 0)
    return fail(B2A_ERR_ALIGN, "%s: the pool and its pages must be 16-byte aligned", who);
  return B2A_OK;
}

Q4::Pool q4_pool_of(const void* pool, int n_pages, int page_rows, long long page_bytes, int D, bool paged_cache) {
  return Q4::Pool{static_cast<unsigned char*>(const_cast<void*>(pool)), page_bytes,
                  paged_cache ? log2_of(page_rows) : -1, page_rows / 16 * Q4::granule_bytes(D), n_pages};
}

}  // namespace

extern "C" {

int b2a_norm_rope_append_paged(const void* q, long long q_tok_stride, const void* k,
                               long long k_tok_stride, const void* v, long long v_tok_stride,
                               int in_dtype, const float* bq, const float* bk, const float* bv,
                               const float* wq, const float* wk, float eps, const float* cos_tab,
                               const float* sin_tab, int tab_rows, const int* pos_dev,
                               const int* slot_dev, void* k_pool, void* v_pool, int n_pages,
                               int page_rows, long long page_stride, int kv_dtype, void* q_out,
                               int n_tok, int H, int KV, int D, int n_rot, int style, void* stream) {
  Q4::AppendArgs a = {q, k, v, q_tok_stride, k_tok_stride, v_tok_stride, bq, bk, bv, wq, wk, cos_tab, sin_tab,
                      pos_dev, slot_dev, k_pool, v_pool, q_out, page_stride,
                      static_cast<long long>(n_pages) * page_rows, D > 0 ? 1.0 / D : 0.0, eps, tab_rows,
                      log2_of(page_rows), H, KV, D, n_rot, style == B2A_ROPE_NEOX ? 1 : 0, n_tok};
  const int rc = norm_append_check("norm_rope_append_paged", a, in_dtype, kv_dtype, n_pages, page_rows, style);
  if (rc) return rc;
  const long long page_elems = static_cast<long long>(page_rows) * KV * D;
  if (a.page_stride == 0) a.page_stride = page_elems;
  if (a.page_stride < page_elems)
    return fail(B2A_ERR_SHAPE, "norm_rope_append_paged: page_stride %lld < page_rows*KV*D %lld", page_stride, page_elems);
  if (a.page_stride * b2a_host::elem_size(kv_dtype) % 16 != 0)
    return fail(B2A_ERR_ALIGN, "norm_rope_append_paged: pages must be 16-byte aligned");
  if (n_tok == 0) return B2A_OK;
  const cudaError_t e = with_type(in_dtype, [&](auto* ts) {
    return with_type(kv_dtype, [&](auto* tk) {
      using TS = typename std::remove_pointer<decltype(ts)>::type;
      using TK = typename std::remove_pointer<decltype(tk)>::type;
      return norm_append_launch<TS, TK, TK, false>(a, static_cast<cudaStream_t>(stream));
    });
  });
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "norm_rope_append_paged launch");
}

int b2a_rope_append_q4(const void* q, long long q_tok_stride, const void* k, long long k_tok_stride,
                       const void* v, long long v_tok_stride, int in_dtype, const float* bq,
                       const float* bk, const float* bv, const float* wq, const float* wk, float eps,
                       const float* cos_tab, const float* sin_tab, int tab_rows, const int* pos_dev,
                       const int* slot_dev, void* pool, int n_pages, int page_rows,
                       long long page_bytes, void* q_out, int q_out_dtype, int n_tok, int H, int KV,
                       int D, int n_rot, int style, void* stream) {
  Q4::AppendArgs a = {q, k, v, q_tok_stride, k_tok_stride, v_tok_stride, bq, bk, bv, wq, wk, cos_tab, sin_tab,
                      pos_dev, slot_dev, pool, pool, q_out, 0,
                      static_cast<long long>(n_pages) * page_rows, D > 0 ? 1.0 / D : 0.0, eps, tab_rows,
                      log2_of(page_rows), H, KV, D, n_rot, style == B2A_ROPE_NEOX ? 1 : 0, n_tok};
  int rc = norm_append_check("rope_append_q4", a, in_dtype, q_out_dtype, n_pages, page_rows, style);
  if (rc == B2A_OK) rc = q4_pool_check("rope_append_q4", pool, n_pages, page_rows, page_bytes, KV, D, true);
  if (rc) return rc;
  if (style == B2A_ROPE_NEOX && n_rot % 64 != 0)
    return fail(B2A_ERR_SHAPE, "rope_append_q4: neox n_rot %d is not a multiple of 64", n_rot);
  if (q_out_dtype == B2A_F32) return fail(B2A_ERR_DTYPE, "rope_append_q4: q_out must be f16 or bf16");
  a.page_stride = page_bytes;
  if (n_tok == 0) return B2A_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(in_dtype, [&](auto* ts) {
    using TS = typename std::remove_pointer<decltype(ts)>::type;
    if (q_out_dtype == B2A_F16) return norm_append_launch<TS, float, __half, true>(a, st);
    return norm_append_launch<TS, float, __nv_bfloat16, true>(a, st);
  });
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "rope_append_q4 launch");
}

int b2a_q4_rows(const void* pool, int n_pages, int page_rows, long long page_bytes, const int* slot_dev,
                void* k_out, void* v_out, int out_dtype, int n_tok, int KV, int D, void* stream) {
  const int rc = q4_pool_check("q4_rows", pool, n_pages, page_rows, page_bytes, KV, D, true);
  if (rc) return rc;
  if (!slot_dev || !k_out || !v_out) return fail(B2A_ERR_ARG, "q4_rows: null pointer argument");
  if (n_tok < 0) return fail(B2A_ERR_ARG, "q4_rows: n_tok %d", n_tok);
  if (b2a_host::elem_size(out_dtype) == 0) return fail(B2A_ERR_DTYPE, "q4_rows: dtype %d", out_dtype);
  if (!b2a_host::aligned16(k_out) || !b2a_host::aligned16(v_out))
    return fail(B2A_ERR_ALIGN, "q4_rows: outputs must be 16-byte aligned");
  if (n_tok == 0) return B2A_OK;
  const Q4::Pool p = q4_pool_of(pool, n_pages, page_rows, page_bytes, D, true);
  const int ctas = n_tok / 8 + (n_tok % 8 != 0);
  const int most = 8 * b2a_host::sm_count();
  const cudaError_t e = with_type(out_dtype, [&](auto* t) {
    using T = typename std::remove_pointer<decltype(t)>::type;
    return b2a_host::launch(Q4::q4_rows_kernel<T>, dim3(ctas < most ? ctas : most),
                            dim3(Q4::kThreads), 0, static_cast<cudaStream_t>(stream), p, slot_dev,
                            static_cast<T*>(k_out), static_cast<T*>(v_out), n_tok, KV, D);
  });
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "q4_rows launch");
}

int b2a_tree_commit_q4(const int* picks_dev, const int* tokens_dev, const int* parents_dev,
                       const int* cu_dev, const int* lens_dev, const int* table_dev,
                       long long table_stride, int table_width, void* pool, int n_layers,
                       long long layer_bytes, int n_pages, int page_rows, long long page_bytes, int KV,
                       int D, int B, int n_tok, int max_nodes, int max_len, int* path_dev,
                       int* accepted_dev, int* next_dev, int* lens_out_dev, void* stream) {
  if ((n_tok > 0 && (!picks_dev || !tokens_dev)) || !cu_dev || !lens_dev || !path_dev || !accepted_dev ||
      !next_dev || !lens_out_dev)
    return fail(B2A_ERR_ARG, "tree_commit_q4: null pointer argument");
  if (n_layers <= 0 || B <= 0 || n_tok < 0 || max_len <= 0)
    return fail(B2A_ERR_ARG, "tree_commit_q4: sizes must be positive");
  if (max_nodes <= 0 || max_nodes > B2A_TREE_MAX_NODES)
    return fail(B2A_ERR_ARG, "tree_commit_q4: max_nodes %d (1..%d)", max_nodes, B2A_TREE_MAX_NODES);
  if (B > 65535) return fail(B2A_ERR_UNSUPPORTED, "tree_commit_q4: %d requests > 65535", B);
  if (lens_out_dev == lens_dev)
    return fail(B2A_ERR_ARG, "tree_commit_q4: lens_out needs a buffer of its own");
  const int rc = q4_pool_check("tree_commit_q4", pool, n_pages, page_rows, page_bytes, KV, D, table_dev != nullptr);
  if (rc) return rc;
  const long long dense = static_cast<long long>(KV) * (page_rows / 16) * Q4::granule_bytes(D);
  if (n_layers > 1 && (layer_bytes < page_bytes * (n_pages - 1) + dense || layer_bytes % 16 != 0))
    return fail(B2A_ERR_SHAPE, "tree_commit_q4: layers overlap or are not 16-byte aligned");
  if (table_dev) {
    if (table_width <= 0 || table_stride < table_width ||
        static_cast<long long>(table_width) * page_rows < max_len)
      return fail(B2A_ERR_SHAPE, "tree_commit_q4: a table row of %d pages (stride %lld) does not hold max_len %d rows",
                  table_width, table_stride, max_len);
  } else if (n_pages < B || page_rows < max_len) {
    return fail(B2A_ERR_SHAPE, "tree_commit_q4: %d blocks of %d rows for %d sequences of up to %d",
                n_pages, page_rows, B, max_len);
  }
  const Q4::Pool p = q4_pool_of(pool, n_pages, page_rows, page_bytes, D, table_dev != nullptr);
  PG::Commit c = {};
  c.picks = picks_dev;
  c.tokens = tokens_dev;
  c.parents = parents_dev;
  c.cu = cu_dev;
  c.lens = lens_dev;
  c.table = table_dev;
  c.table_stride = table_stride;
  c.layer_bytes = n_layers > 1 ? layer_bytes : 0;
  c.n_layers = n_layers;
  c.n_pages = n_pages;
  c.page_shift = p.page_shift;
  c.max_len = max_len;
  c.n_tok = n_tok;
  c.max_nodes = max_nodes;
  c.path = path_dev;
  c.accepted = accepted_dev;
  c.next = next_dev;
  c.lens_out = lens_out_dev;
  const long long cols = static_cast<long long>(n_layers) * KV * (D / 8);
  const long long gx = (cols + PG::kCommitThreads - 1) / PG::kCommitThreads;
  const cudaError_t e = b2a_host::launch(Q4::tree_commit_q4_kernel, dim3(static_cast<unsigned>(gx < 64 ? gx : 64), B),
                                         dim3(PG::kCommitThreads), 0, static_cast<cudaStream_t>(stream), c, p, KV, D);
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "tree_commit_q4 launch");
}

}  // extern "C"
