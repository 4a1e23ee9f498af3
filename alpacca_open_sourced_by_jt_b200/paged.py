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
of bounds are recorded (`_lib.device_error`).  A call runs on the current stream,
or on `stream` (a torch.cuda.Stream or a raw handle), which its new outputs then
belong to.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from . import _lib, device
from .device import _code

MAX_NODES = 128      # B2A_TREE_MAX_NODES
MAX_REQUESTS = 2048  # B2A_PLAN_MAX_REQUESTS


def _bad(msg: str):
    raise _lib.B2AShapeError(_lib.ERR_SHAPE, msg)


# The checks below run before every launch of a serving step: messages are
# only built when a check fails.

def _i32(name: str, t: torch.Tensor, n: int | None = None):
    if t.dtype is not torch.int32 or not t.is_cuda or not t.is_contiguous() or (
            n is not None and t.numel() != n):
        _bad(f"{name} must be a contiguous CUDA int32 tensor" + ("" if n is None else f" of {n}"))


def _i32_rows(name: str, t: torch.Tensor | None, n: int):
    """The address of a per-node array that covers n rows (None: a null pointer)."""
    if t is None:
        return None
    if t.dtype is not torch.int32 or not t.is_cuda or not t.is_contiguous() or t.numel() < n:
        _bad(f"{name} must be a contiguous CUDA int32 tensor of at least {n}")
    return t.data_ptr()


def _f32(name: str, t: torch.Tensor | None, n: int):
    """The address of an f32 array of n (None: a null pointer)."""
    if t is None:
        return None
    if t.dtype is not torch.float32 or not t.is_cuda or not t.is_contiguous() or t.numel() != n:
        _bad(f"{name} must be a contiguous CUDA f32 tensor of {n}")
    return t.data_ptr()


def _table(table, B: int):
    """(address, stride, width) of a block table (B, max_pages), rows of unit stride."""
    if table is None:
        return None, 0, 0
    shape, stride = table.shape, table.stride()
    if table.dtype is not torch.int32 or not table.is_cuda or len(shape) != 2 or shape[0] != B or (
            stride[1] != 1):
        _bad("table must be a CUDA int32 tensor (B, max_pages)")
    return table.data_ptr(), (stride[0] if B > 1 else shape[1]), shape[1]


def _pool(k: torch.Tensor, v: torch.Tensor, dims: int = 4):
    """(shape, strides) of a K and V pool, (n_pages, page_rows, KV, D) with
    contiguous pages; dims 5: (L, ...), a layer stride in front."""
    shape, stride = k.shape, k.stride()
    if not k.is_cuda or not v.is_cuda or len(shape) != dims or v.shape != shape or (
            v.dtype is not k.dtype or v.stride() != stride):
        _bad("k and v pools (n_pages, page_rows, KV, D) of one type and layout")
    R, KV, D = shape[-3:]
    if stride[-1] != 1 or stride[-2] != D or (R > 1 and stride[-3] != KV * D):
        _bad("each page must be contiguous")
    return shape, stride


def _stream(t: torch.Tensor):
    """The current stream of t's device (its raw handle: a torch.cuda.Stream
    object costs microseconds a call)."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _on(stream):
    """A call's `stream` as the current one: what the call allocates then belongs
    to the stream that uses it, and a workspace given back at the call's end is
    not handed to another stream while the kernel still runs."""
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream))
    return torch.cuda.stream(stream)


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
    request, 0 leaves it as it is), pages held.  lens is not written: set an
    ended request's to 0 before its place goes to a new one.  table (B,
    max_pages) and ring (pages of the pool) are updated in place; ring_state (2,) int32 is (head, count) of the free
    pages in the ring.  parents (max_tokens,) gives tree nodes their depth's
    position, None a chain's.  A request the ring cannot serve keeps its pages;
    its tokens' slots and the table entries of the pages it wanted are -1, and
    tree_decode and tree_commit leave it out of the step."""
    if stream is not None:
        with _on(stream):
            return page_plan(lens, add, held, table, ring, ring_state, page_rows=page_rows,
                             max_tokens=max_tokens, parents=parents, out=out)
    B = lens.numel()
    _i32("lens", lens)
    _i32("add", add, B)
    _i32("held", held, B)
    _i32("ring", ring)
    _i32("ring_state", ring_state, 2)
    tptr, tstride, width = _table(table, B)
    if parents is not None:
        _i32("parents", parents, max_tokens)
    if out is None:
        seq, pos, slots, cu, held_out, state_out = torch.empty(
            3 * max_tokens + 2 * B + 3, dtype=torch.int32, device=lens.device).split_with_sizes(
                (max_tokens, max_tokens, max_tokens, B + 1, B, 2))
        out = PagePlan(cu, seq, pos, slots, held_out, state_out)
    else:
        cu, seq, pos, slots, held_out, state_out = out
        _i32("out.cu", cu, B + 1)
        for name, t in (("seq", seq), ("positions", pos), ("slots", slots)):
            _i32("out." + name, t, max_tokens)
        _i32("out.held", held_out, B)
        _i32("out.ring_state", state_out, 2)
    _lib.check(_lib.load().b2a_page_plan(
        lens.data_ptr(), add.data_ptr(), None if parents is None else parents.data_ptr(),
        held.data_ptr(), held_out.data_ptr(), tptr, tstride, ring.data_ptr(), ring.numel(),
        ring_state.data_ptr(), state_out.data_ptr(), cu.data_ptr(), seq.data_ptr(), pos.data_ptr(),
        slots.data_ptr(), B, max_tokens, width, page_rows, _stream(lens)))
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
    if stream is not None:
        with _on(stream):
            return rope_append(q, k, v, positions, slots, cos_tab, sin_tab, k_pool=k_pool,
                               v_pool=v_pool, n_rot=n_rot, style=style, q_out=q_out, bq=bq, bk=bk,
                               bv=bv)
    (P, R, KV, D), pstride = _pool(k_pool, v_pool)
    dt, qs, ks, vs = q.dtype, q.stride(), k.stride(), v.stride()
    n, H, Dq = q.shape
    if not (q.is_cuda and k.is_cuda and v.is_cuda and k.dtype is dt and v.dtype is dt and
            Dq == D and k.shape == (n, KV, D) and v.shape == (n, KV, D)):
        _bad("q (n, H, D), k and v (n, KV, D): CUDA tensors of one type, as the pools' rows")
    if qs[2] != 1 or qs[1] != D or ks[2] != 1 or ks[1] != D or vs[2] != 1 or vs[1] != D:
        _bad("q, k and v rows must be contiguous per token")
    _i32("positions", positions, n)
    _i32("slots", slots, n)
    rows, half = cos_tab.shape
    if n_rot is None:
        n_rot = 2 * half
    if half * 2 != n_rot:
        _bad("cos/sin tables f32 (rows, n_rot/2)")
    cos, sin = _f32("cos_tab", cos_tab, rows * half), _f32("sin_tab", sin_tab, rows * half)
    if q_out is None:
        q_out = k_pool.new_empty((n, H, D))
    elif not q_out.is_cuda or not q_out.is_contiguous() or q_out.numel() != n * H * D:
        _bad("q_out must be a contiguous CUDA tensor (n, H, D)")
    if n == 0:  # (an empty tensor has no address)
        return q_out
    _lib.check(_lib.load().b2a_rope_append_paged(
        q.data_ptr(), qs[0] if n > 1 else H * D, k.data_ptr(), ks[0] if n > 1 else KV * D,
        v.data_ptr(), vs[0] if n > 1 else KV * D, _code(dt), _f32("bq", bq, H * D),
        _f32("bk", bk, KV * D), _f32("bv", bv, KV * D), cos, sin, rows, positions.data_ptr(),
        slots.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), P, R,
        pstride[0] if P > 1 else R * KV * D, _code(k_pool.dtype), q_out.data_ptr(),
        _code(q_out.dtype), n, H, KV, D, n_rot, device._STYLE[style], _stream(q)))
    return q_out


@functools.lru_cache(maxsize=256)
def _tree_bytes(device_index, max_nodes, n_head, n_kv, head_dim, code, max_len) -> int:
    return _lib.load().b2a_tree_decode_workspace_bytes(max_nodes, n_head, n_kv, head_dim, code, max_len)


@functools.lru_cache(maxsize=256)
def _logits_bytes(n_rows, vocab) -> int:
    return _lib.load().b2a_constrain_logits_workspace_bytes(n_rows, vocab)


def tree_decode_workspace(max_nodes: int, n_head: int, n_kv: int, head_dim: int,
                          dtype: torch.dtype, max_len: int, dev) -> torch.Tensor:
    """Allocate (via torch) a workspace big enough for b2a_tree_decode."""
    n = _lib.load().b2a_tree_decode_workspace_bytes(max_nodes, n_head, n_kv, head_dim, _code(dtype),
                                                    max_len)
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
    Returns out (n, H, D) in q's type, padding rows and those of requests left
    out zero; lse (n, H) f32 receives the natural-log log-sum-exp if given."""
    if stream is not None:
        with _on(stream):
            return tree_decode(q, k_pool, v_pool, lens, cu, parents, table=table,
                               max_nodes=max_nodes, max_len=max_len, scale=scale, out=out, lse=lse,
                               workspace=workspace)
    (P, R, KV, D), pstride = _pool(k_pool, v_pool)
    dt, qs = q.dtype, q.stride()
    n, H, Dq = q.shape
    if not q.is_cuda or qs[2] != 1 or qs[1] != D or Dq != D or k_pool.dtype is not dt:
        _bad("q must be a CUDA tensor (n, H, D), contiguous per token, in the pools' type")
    B = lens.numel()
    _i32("lens", lens)
    _i32("cu", cu, B + 1)
    pptr = _i32_rows("parents", parents, n)
    tptr, tstride, width = _table(table, B)
    if max_len is None:
        max_len = width * R if table is not None else R
    if out is None:
        out = q.new_empty((n, H, D))
    elif not out.is_cuda or not out.is_contiguous() or out.shape != (n, H, D) or out.dtype is not dt:
        _bad("out must be a contiguous CUDA tensor (n, H, D) in q's type")
    if n == 0:
        return out
    lib = _lib.load()
    code = _code(dt)
    if workspace is None:
        ws_bytes = _tree_bytes(q.device.index, max_nodes, H, KV, D, code, max_len)
        # (held until the launch below: the allocator hands it out again in stream order)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    else:
        ws_bytes = workspace.numel() * workspace.element_size()
    _lib.check(lib.b2a_tree_decode(
        q.data_ptr(), qs[0] if n > 1 else H * D, k_pool.data_ptr(), v_pool.data_ptr(), P, R,
        pstride[0] if P > 1 else R * KV * D, tptr, tstride, width, lens.data_ptr(), cu.data_ptr(),
        pptr, out.data_ptr(), _f32("lse", lse, n * H),
        None if workspace is None else workspace.data_ptr(), ws_bytes, B, n,
        max_nodes, H, KV, D, code, 1.0 / math.sqrt(D) if scale is None else scale, max_len,
        _stream(q)))
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
    if stream is not None:
        with _on(stream):
            return constrain_logits(
                logits, cu, parents, tokens, max_nodes=max_nodes, hist=hist, hist_start=hist_start,
                prompt_lens=prompt_lens, repetition=repetition, presence=presence,
                frequency=frequency, bias_start=bias_start, bias_ids=bias_ids, bias=bias, mask=mask,
                out=out, picks=picks, workspace=workspace)
    n, V = logits.shape
    ls = logits.stride()
    if not logits.is_cuda or ls[1] != 1:
        _bad("logits must be a CUDA tensor (n, V), unit stride along V")
    B = cu.numel() - 1
    _i32("cu", cu)
    n_hist = n_bias = mstride = 0
    hptr = sptr = bsptr = biptr = mptr = None
    if hist is not None:
        if hist_start is None:
            _bad("hist needs hist_start")
        n_hist = hist.numel()
        hptr, sptr = _i32_rows("hist", hist, 0), _i32_rows("hist_start", hist_start, B + 1)
    if bias is not None:
        if bias_start is None or bias_ids is None:
            _bad("bias needs bias_start and bias_ids")
        n_bias = bias.numel()
        bsptr, biptr = _i32_rows("bias_start", bias_start, B + 1), _i32_rows("bias_ids", bias_ids, n_bias)
    if mask is not None:
        mshape, mstride = mask.shape, mask.stride()
        if mask.dtype not in (torch.int32, torch.uint32) or not mask.is_cuda or len(mshape) != 2 or (
                mshape[0] != n or mstride[1] != 1 or mshape[1] * 32 < V):
            _bad("mask must be a CUDA int32 tensor (n, V / 32) of words")
        mptr, mstride = mask.data_ptr(), (mstride[0] if n > 1 else mshape[1])
    if out is None:
        out = torch.empty((n, V), dtype=torch.float32, device=logits.device)
    os = out.stride()
    if not out.is_cuda or out.shape != (n, V) or os[1] != 1:
        _bad("out must be a CUDA tensor (n, V), unit stride along V")
    lib = _lib.load()
    if workspace is None:
        ws_bytes = _logits_bytes(n, V)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=logits.device)
    else:
        ws_bytes = workspace.numel() * workspace.element_size()
    if picks is None:
        picks = torch.empty(n, dtype=torch.int32, device=logits.device)
    else:
        _i32("picks", picks, n)
    if n == 0:
        return out, picks
    _lib.check(lib.b2a_constrain_logits(
        logits.data_ptr(), ls[0] if n > 1 else V, _code(logits.dtype), out.data_ptr(),
        os[0] if n > 1 else V, _code(out.dtype), picks.data_ptr(), cu.data_ptr(),
        _i32_rows("parents", parents, n), _i32_rows("tokens", tokens, n), hptr, sptr, n_hist,
        _i32_rows("prompt_lens", prompt_lens, B), _f32("repetition", repetition, B),
        _f32("presence", presence, B), _f32("frequency", frequency, B), bsptr, biptr,
        _f32("bias", bias, n_bias), n_bias, mptr, mstride, B, n, max_nodes, V,
        workspace.data_ptr(), ws_bytes, _stream(logits)))
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
    (L, B, n_ctx, KV, D) blocks).  A request left out (page_plan could not serve
    it) has accepted 0, next_token -1, its lens as it was, and moves no rows."""
    if stream is not None:
        with _on(stream):
            return tree_commit(picks, tokens, parents, cu, lens, k_pool, v_pool, table=table,
                               max_nodes=max_nodes, max_len=max_len, out=out)
    dims = k_pool.dim()
    shape, strides = _pool(k_pool, v_pool, 5 if dims == 5 else 4)
    P, R, KV, D = shape[-4:]
    L = shape[0] if dims == 5 else 1
    B, n = lens.numel(), tokens.numel()
    _i32("lens", lens)
    _i32("cu", cu, B + 1)
    tptr, tstride, width = _table(table, B)
    if max_len is None:
        max_len = width * R if table is not None else R
    if out is None:
        path, accepted, nxt, lens_out = torch.empty(
            B * (max_nodes + 3), dtype=torch.int32,
            device=lens.device).split_with_sizes((B * max_nodes, B, B, B))
        out = Commit(path.view(B, max_nodes), accepted, nxt, lens_out)
    else:
        path, accepted, nxt, lens_out = out
        _i32("out.path", path, B * max_nodes)
        for name, t in (("accepted", accepted), ("next_token", nxt), ("lens", lens_out)):
            _i32("out." + name, t, B)
    _lib.check(_lib.load().b2a_tree_commit(
        _i32_rows("picks", picks, n), _i32_rows("tokens", tokens, n),
        _i32_rows("parents", parents, n), cu.data_ptr(), lens.data_ptr(), tptr, tstride, width,
        k_pool.data_ptr(), v_pool.data_ptr(), L, strides[0] if L > 1 else 0, P, R,
        strides[-4] if P > 1 else R * KV * D, KV, D, _code(k_pool.dtype), B, n, max_nodes, max_len,
        path.data_ptr(), accepted.data_ptr(), nxt.data_ptr(), lens_out.data_ptr(),
        _stream(lens)))
    return out
