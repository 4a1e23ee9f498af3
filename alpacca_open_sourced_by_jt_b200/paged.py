"""Many requests over one paged KV cache, with trees of drafted tokens:
device-tensor API over libb2attn.so.

A step of a serving loop:

    plan  = page_plan(lens, add, held, table, ring, ring_state, ...)
    per layer:
      qr  = rope_append(q, k, v, plan.positions, plan.slots, cos, sin, k_pool=..., v_pool=...)
      att = tree_decode(qr, k_pool, v_pool, lens, plan.cu, parents, table=table, ...)
    logits, picks = constrain_logits(logits, plan.cu, parents, tokens, ...)
    done  = tree_commit(picks, tokens, parents, plan.cu, lens, k_pools, v_pools, table=table, ...)

Pools are (n_pages, page_rows, KV, D) tensors and `table` (B, max_pages) int32
names each request's pages; page_rows is a power of two.  The step's tokens
(nodes) of all requests lie behind one another: request b owns rows cu[b] ..
cu[b + 1] - 1.  `parents` holds each node's parent as an index inside its
request (-1: a root), or is None for chains; a request has at most
MAX_NODES nodes.  Rows from cu[B] on are padding (captured steps).

As in `device`, every function checks its arguments on the host, makes one
C-ABI call and never synchronises; numbers that live on the device and are out
of bounds are recorded (`_lib.device_error`).
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib, device
from .device import _code, _need, _ptr, _stream

MAX_NODES = 128      # B2A_TREE_MAX_NODES
MAX_REQUESTS = 2048  # B2A_PLAN_MAX_REQUESTS


def _i32(name: str, t: torch.Tensor, n: int | None = None):
    _need(t.dtype == torch.int32 and t.is_cuda and t.is_contiguous() and
          (n is None or t.numel() == n),
          f"{name} must be a contiguous CUDA int32 tensor" + (f" of {n}" if n is not None else ""))


def _table(table, B: int):
    """(stride, width) of a block table (B, max_pages), rows of unit stride."""
    if table is None:
        return 0, 0
    _need(table.dtype == torch.int32 and table.is_cuda and table.dim() == 2 and
          table.shape[0] == B and table.stride(1) == 1,
          "table must be a CUDA int32 tensor (B, max_pages)")
    return (table.stride(0) if B > 1 else table.shape[1]), table.shape[1]


def _pool(k: torch.Tensor, v: torch.Tensor):
    """(n_pages, page_rows, page_stride, KV, D) of a K and V pool."""
    _need(k.is_cuda and v.is_cuda and k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and
          k.stride() == v.stride(), "k and v pools (n_pages, page_rows, KV, D) of one type and layout")
    P, R, KV, D = k.shape
    _need(k[0].is_contiguous(), "each page must be contiguous")
    return P, R, (k.stride(0) if P > 1 else R * KV * D), KV, D


class PagePlan(NamedTuple):
    """What page_plan leaves: cu (B + 1), seq / positions / slots (max_tokens),
    and the numbers of the next step: held (B), ring_state (2)."""
    cu: torch.Tensor
    seq: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    held: torch.Tensor
    ring_state: torch.Tensor


def page_plan(lens: torch.Tensor, add: torch.Tensor, held: torch.Tensor, table: torch.Tensor,
              ring: torch.Tensor, ring_state: torch.Tensor, *, page_rows: int, max_tokens: int,
              parents: torch.Tensor | None = None, out: PagePlan | None = None,
              stream=None) -> PagePlan:
    """Block tables, slot map and positions of a step, on the device
    (b2a_page_plan).

    lens, add, held (B,) int32: cached rows, tokens to add (-1 ends the
    request), pages held.  table (B, max_pages) and ring (pages of the pool)
    are updated in place; ring_state (2,) int32 is (head, count) of the free
    pages in the ring.  parents (max_tokens,) gives tree nodes their depth's
    position, None a chain's.  A request the ring cannot serve keeps its pages
    and its tokens' slots are -1."""
    B = lens.numel()
    _i32("lens", lens)
    _i32("add", add, B)
    _i32("held", held, B)
    _i32("ring", ring)
    _i32("ring_state", ring_state, 2)
    stride, width = _table(table, B)
    if parents is not None:
        _i32("parents", parents, max_tokens)
    if out is None:
        # one allocation: five int32 arrays, the three per-token ones 16-byte aligned
        n = (max_tokens + 3) & ~3
        buf = torch.empty(3 * n + 2 * B + 3, dtype=torch.int32, device=lens.device)
        out = PagePlan(buf[3 * n:3 * n + B + 1], buf[:max_tokens], buf[n:n + max_tokens],
                       buf[2 * n:2 * n + max_tokens], buf[3 * n + B + 1:3 * n + 2 * B + 1],
                       buf[3 * n + 2 * B + 1:])
    else:
        _i32("out.cu", out.cu, B + 1)
        for name, t in (("seq", out.seq), ("positions", out.positions), ("slots", out.slots)):
            _i32("out." + name, t, max_tokens)
        _i32("out.held", out.held, B)
        _i32("out.ring_state", out.ring_state, 2)
    _lib.check(_lib.load().b2a_page_plan(
        _ptr(lens), _ptr(add), _ptr(parents), _ptr(held), _ptr(out.held), _ptr(table), stride,
        _ptr(ring), ring.numel(), _ptr(ring_state), _ptr(out.ring_state), _ptr(out.cu),
        _ptr(out.seq), _ptr(out.positions), _ptr(out.slots), B, int(max_tokens), width,
        int(page_rows), _stream(stream)))
    return out


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                slots: torch.Tensor, cos_tab: torch.Tensor, sin_tab: torch.Tensor, *, k_pool,
                v_pool, n_rot: int | None = None, style: str = "norm", q_out=None, bq=None,
                bk=None, bv=None, stream=None) -> torch.Tensor:
    """Fused bias + RoPE + append into a paged cache (b2a_rope_append_paged).

    q (n, H, D), k, v (n, KV, D) of one type (f32, f16 or bf16), contiguous per
    token (views into one packed projection are fine); positions, slots (n,)
    int32 as page_plan writes them: the rotary position and the pool row are
    apart, a negative slot stores nothing.  Returns q_out (n, H, D), in the
    pools' type unless given."""
    _need(q.dim() == 3 and k.dim() == 3 and k.shape == v.shape and q.dtype == k.dtype == v.dtype and
          q.is_cuda and k.is_cuda and v.is_cuda, "q (n,H,D), k/v (n,KV,D) CUDA tensors of one type")
    n, H, D = q.shape
    P, R, pstride, KV, Dp = _pool(k_pool, v_pool)
    _need(k.shape == (n, KV, D) and Dp == D, "k/v rows do not match the pools")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _need(t.stride(2) == 1 and t.stride(1) == D, f"{name} rows must be contiguous per token")
    _i32("positions", positions, n)
    _i32("slots", slots, n)
    device._cuda_contig("cos_tab", cos_tab)
    device._cuda_contig("sin_tab", sin_tab)
    if n_rot is None:
        n_rot = 2 * cos_tab.shape[1]
    _need(cos_tab.shape == sin_tab.shape and cos_tab.shape[1] * 2 == n_rot and
          cos_tab.dtype == sin_tab.dtype == torch.float32, "cos/sin tables f32 (rows, n_rot/2)")
    for name, t, m in (("bq", bq, H), ("bk", bk, KV), ("bv", bv, KV)):
        if t is not None:
            device._cuda_contig(name, t)
            _need(t.dtype == torch.float32 and t.numel() == m * D, f"{name} f32 ({m}, D)")
    if q_out is None:
        q_out = torch.empty((n, H, D), dtype=k_pool.dtype, device=q.device)
    else:
        device._cuda_contig("q_out", q_out)
        _need(q_out.numel() == n * H * D, "q_out (n, H, D)")

    def stride(t, m):
        return t.stride(0) if n > 1 else m * D

    _lib.check(_lib.load().b2a_rope_append_paged(
        _ptr(q), stride(q, H), _ptr(k), stride(k, KV), _ptr(v), stride(v, KV), _code(q.dtype),
        _ptr(bq), _ptr(bk), _ptr(bv), _ptr(cos_tab), _ptr(sin_tab), cos_tab.shape[0],
        _ptr(positions), _ptr(slots), _ptr(k_pool), _ptr(v_pool), P, R, pstride,
        _code(k_pool.dtype), _ptr(q_out), _code(q_out.dtype), n, H, KV, D, int(n_rot),
        device._STYLE[style], _stream(stream)))
    return q_out


def tree_decode_workspace(max_nodes: int, n_head: int, n_kv: int, head_dim: int,
                          dtype: torch.dtype, dev) -> torch.Tensor:
    """Allocate (via torch) a workspace big enough for b2a_tree_decode."""
    n = _lib.load().b2a_tree_decode_workspace_bytes(max_nodes, n_head, n_kv, head_dim, _code(dtype))
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device=dev)


def tree_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, lens: torch.Tensor,
                cu: torch.Tensor, parents: torch.Tensor | None, *, table=None, max_nodes: int,
                max_len: int | None = None, scale: float | None = None, out=None, lse=None,
                workspace=None, stream=None) -> torch.Tensor:
    """Attention of drafted tokens over the cache (b2a_tree_decode).

    q (n, H, D) in the pools' type; pools (n_pages, page_rows, KV, D) with
    table (B, max_pages), or, with table None, one block per sequence (B,
    n_ctx, KV, D).  lens (B,) int32 cached rows before the tree; cu (B + 1,)
    and parents (n,) the trees (None: chains).  Node i reads the cached rows,
    its ancestors' rows and its own, which stand at rows lens[b] + node.
    max_len bounds lens + nodes (default: what the table or the block holds).
    Returns out (n, H, D) in q's type, padding rows zero; lse (n, H) f32
    receives the natural-log log-sum-exp if given."""
    _need(q.dim() == 3 and q.is_cuda and q.stride(2) == 1 and q.stride(1) == q.shape[2],
          "q must be a CUDA tensor (n, H, D), contiguous per token")
    n, H, D = q.shape
    P, R, pstride, KV, Dp = _pool(k_pool, v_pool)
    _need(Dp == D and k_pool.dtype == q.dtype, "the pools must have q's head_dim and type")
    B = lens.numel()
    _i32("lens", lens)
    _i32("cu", cu, B + 1)
    if parents is not None:
        _i32("parents", parents)
        _need(parents.numel() >= n, "parents must cover q's rows")
    tstride, width = _table(table, B)
    if max_len is None:
        max_len = width * R if table is not None else R
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((n, H, D), dtype=q.dtype, device=q.device)
    else:
        device._cuda_contig("out", out)
        _need(out.shape == (n, H, D) and out.dtype == q.dtype, "out (n, H, D) in q's type")
    if lse is not None:
        device._cuda_contig("lse", lse)
        _need(lse.dtype == torch.float32 and lse.numel() == n * H, "lse must be f32 (n, H)")
    if workspace is None:
        workspace = tree_decode_workspace(max_nodes, H, KV, D, q.dtype, q.device)
    _lib.check(_lib.load().b2a_tree_decode(
        _ptr(q), q.stride(0) if n > 1 else H * D, _ptr(k_pool), _ptr(v_pool), P, R, pstride,
        _ptr(table), tstride, width, _ptr(lens), _ptr(cu), _ptr(parents), _ptr(out), _ptr(lse),
        _ptr(workspace), workspace.numel() * workspace.element_size(), B, n, int(max_nodes), H, KV,
        D, _code(q.dtype), float(scale), int(max_len), _stream(stream)))
    return out


def constrain_logits(logits: torch.Tensor, cu: torch.Tensor, parents: torch.Tensor | None,
                     tokens: torch.Tensor | None, *, max_nodes: int, hist=None, hist_start=None,
                     prompt_lens=None, repetition=None, presence=None, frequency=None,
                     bias_start=None, bias_ids=None, bias=None, mask=None, out=None, picks=None,
                     workspace=None, stream=None):
    """Penalties for repeated tokens, biases and grammar masks on logits rows,
    and each row's greedy pick (b2a_constrain_logits).

    logits (n, V) f32, f16 or bf16, unit stride along V: one row per node; cu,
    parents, tokens the trees and their tokens (tokens None: a node's path is
    not counted).  hist int32 holds the requests' tokens behind one another,
    request b's at hist_start[b] .. hist_start[b + 1], its first
    prompt_lens[b] the prompt.  repetition / presence / frequency (B,) f32 or
    None.  bias_ids int32 and bias f32 hold the requests' (token, bias) entries
    behind one another, bias_start (B + 1,) their starts.  mask (n, >= V / 32)
    int32: bit v % 32 of word v / 32 allows token v.  Returns (out, picks): out
    defaults to a new f32 tensor (pass out=logits for in place); picks (n,)
    int32, -1 where nothing can be picked."""
    _need(logits.dim() == 2 and logits.is_cuda and logits.stride(1) == 1, "logits CUDA (n, V)")
    n, V = logits.shape
    B = cu.numel() - 1
    _i32("cu", cu)
    for name, t in (("parents", parents), ("tokens", tokens)):
        if t is not None:
            _i32(name, t)
            _need(t.numel() >= n, f"{name} must cover the rows")
    if hist is not None:
        _i32("hist", hist)
        _need(hist_start is not None, "hist needs hist_start")
        _i32("hist_start", hist_start, B + 1)
    if prompt_lens is not None:
        _i32("prompt_lens", prompt_lens, B)
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None:
            device._cuda_contig(name, t)
            _need(t.dtype == torch.float32 and t.numel() == B, f"{name} f32 (B,)")
    if bias is not None:
        _need(bias_start is not None and bias_ids is not None, "bias needs bias_start and bias_ids")
        _i32("bias_start", bias_start, B + 1)
        _i32("bias_ids", bias_ids, bias.numel())
        device._cuda_contig("bias", bias)
        _need(bias.dtype == torch.float32, "bias f32")
    if mask is not None:
        _need(mask.dtype in (torch.int32, torch.uint32) and mask.is_cuda and mask.dim() == 2 and
              mask.shape[0] == n and mask.stride(1) == 1 and mask.shape[1] * 32 >= V,
              "mask int32 (n, V / 32) words")
    if out is None:
        out = torch.empty((n, V), dtype=torch.float32, device=logits.device)
    _need(out.shape == (n, V) and out.is_cuda and out.stride(1) == 1, "out CUDA (n, V)")
    if picks is None:
        picks = torch.empty(n, dtype=torch.int32, device=logits.device)
    else:
        _i32("picks", picks, n)
    lib = _lib.load()
    if workspace is None:
        workspace = torch.empty(max(lib.b2a_constrain_logits_workspace_bytes(n, V), 16),
                                dtype=torch.uint8, device=logits.device)

    def stride(t, w):
        return t.stride(0) if n > 1 else w

    _lib.check(lib.b2a_constrain_logits(
        _ptr(logits), stride(logits, V), _code(logits.dtype), _ptr(out), stride(out, V),
        _code(out.dtype), _ptr(picks), _ptr(cu), _ptr(parents), _ptr(tokens), _ptr(hist),
        _ptr(hist_start), 0 if hist is None else hist.numel(), _ptr(prompt_lens),
        _ptr(repetition), _ptr(presence), _ptr(frequency), _ptr(bias_start), _ptr(bias_ids),
        _ptr(bias), 0 if bias is None else bias.numel(), _ptr(mask),
        0 if mask is None else stride(mask, mask.shape[1]), B, n, int(max_nodes), V,
        _ptr(workspace), workspace.numel() * workspace.element_size(), _stream(stream)))
    return out, picks


class Commit(NamedTuple):
    """What tree_commit leaves: path (B, max_nodes) node indices, -1 behind;
    accepted (B,); next_token (B,); lens (B,), the cached rows after it."""
    path: torch.Tensor
    accepted: torch.Tensor
    next_token: torch.Tensor
    lens: torch.Tensor


def tree_commit(picks: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor | None,
                cu: torch.Tensor, lens: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                *, table=None, max_nodes: int, max_len: int | None = None, out: Commit | None = None,
                stream=None) -> Commit:
    """The accepted path of each tree, its K/V rows moved into place
    (b2a_tree_commit).

    picks, tokens (n,) int32: the model's token after each node and the node's
    own.  Pools (L, n_pages, page_rows, KV, D) for all layers at once, or one
    layer's 4-D pool; table, lens, cu, parents as in tree_decode (table None:
    (L, B, n_ctx, KV, D) blocks)."""
    if k_pool.dim() == 4:
        k_pool, v_pool = k_pool.unsqueeze(0), v_pool.unsqueeze(0)
    _need(k_pool.dim() == 5 and k_pool.shape == v_pool.shape and k_pool.stride() == v_pool.stride(),
          "pools (L, n_pages, page_rows, KV, D)")
    L = k_pool.shape[0]
    P, R, pstride, KV, D = _pool(k_pool[0], v_pool[0])
    B, n = lens.numel(), tokens.numel()
    _i32("lens", lens)
    _i32("cu", cu, B + 1)
    _i32("tokens", tokens)
    _i32("picks", picks)
    _need(picks.numel() >= n, "picks must cover the tokens")
    if parents is not None:
        _i32("parents", parents)
        _need(parents.numel() >= n, "parents must cover the tokens")
    tstride, width = _table(table, B)
    if max_len is None:
        max_len = width * R if table is not None else R
    if out is None:
        buf = torch.empty(B * (max_nodes + 3), dtype=torch.int32, device=lens.device)
        m = B * max_nodes
        out = Commit(buf[:m].view(B, max_nodes), buf[m:m + B], buf[m + B:m + 2 * B], buf[m + 2 * B:])
    else:
        _i32("out.path", out.path, B * max_nodes)
        for name, t in (("accepted", out.accepted), ("next_token", out.next_token), ("lens", out.lens)):
            _i32("out." + name, t, B)
    _lib.check(_lib.load().b2a_tree_commit(
        _ptr(picks), _ptr(tokens), _ptr(parents), _ptr(cu), _ptr(lens), _ptr(table), tstride, width,
        _ptr(k_pool), _ptr(v_pool), L, k_pool.stride(0) if L > 1 else 0, P, R, pstride, KV, D,
        _code(k_pool.dtype), B, n, int(max_nodes), int(max_len), _ptr(out.path), _ptr(out.accepted),
        _ptr(out.next_token), _ptr(out.lens), _stream(stream)))
    return out
