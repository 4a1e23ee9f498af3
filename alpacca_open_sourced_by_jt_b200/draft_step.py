"""Many requests of one Q8_0 llama model over a paged cache, verifying trees of
drafted tokens: the path that runs the operators of `paged` as they are used.

The reference serves one sequence per Model, a token per step
(Model._forward_np, alpaccaroo/model.py:1374-1487).  Here a step takes, for
each request, a tree of drafted tokens whose root is the request's last token,
evaluates all nodes of all requests at once, and keeps the longest path that
the model itself would have picked:

  plan                   b2a_page_plan: pages, slots and positions of the nodes
  embed rows             b2a_q8_embed
  per layer:
    h    = RMSNorm(x)    b2a_rmsnorm_rows (the cache's 16-bit type)
    qkv  = h . Wqkv^T    b2a_gemm, f32 rows
    RoPE, K/V rows to their slots, q to 16 bits   b2a_rope_append_paged
    att  = the nodes over the cache               b2a_tree_decode
      (models that norm their heads: b2a_norm_rope_append_paged; a cache of 4
      bits: b2a_rope_append_q4, b2a_tree_decode_q4)
    x   += att . Wo^T    b2a_gemm, in place
    act  = SwiGLU(RMSNorm(x) . Wgu^T)             b2a_gemm
    x   += act . Wdown^T b2a_gemm, in place
  logits = RMSNorm(x) . Woutput^T                 b2a_gemm_q8
  penalties, biases, masks, picks                 b2a_constrain_logits
  where tokens are sampled, which drafts stand    b2a_verify_picks (the former then
                                                  only for limits)
  accepted paths, K/V rows into place             b2a_tree_commit, b2a_tree_commit_q4

Prompts go through the same layers in chunks, as chains.  Where the drafts
come from is the caller's (an n-gram table, a small model)."""
from __future__ import annotations

import torch

from . import _lib, device, paged
from .decode_chain import LlamaQ8
from .prefill_chain import ChunkPrefill, _dequant


class DraftStep:
    """`requests` slots over a pool of n_pages pages of page_rows rows per
    layer, at most max_len rows a request (prompts and trees that pass it are
    refused).  dtype (f16 or bf16) is the 16-bit operands'; kv_bits 16: the
    cache's too, 4: the cache holds blocks of 32 values with a scale
    (paged.q4_pool)."""

    def __init__(self, model: LlamaQ8, requests: int, n_pages: int, *, page_rows: int = 64,
                 max_len: int = 4096, dtype: torch.dtype = torch.float16, kv_bits: int = 16):
        _lib.load()
        if dtype not in (torch.float16, torch.bfloat16):
            raise _lib.B2AShapeError(_lib.ERR_DTYPE, "the paged cache must be f16 or bf16")
        if kv_bits not in (4, 16):
            raise _lib.B2AShapeError(_lib.ERR_ARG, f"kv_bits {kv_bits} (4 or 16)")
        if model.F % 128:
            raise _lib.B2AShapeError(_lib.ERR_SHAPE, "16-bit GEMMs need n_ff % 128 == 0")
        m, dev = model, model.device
        self.m, self.dt, self.B, self.page_rows, self.max_len = m, dtype, requests, page_rows, max_len
        i32 = dict(dtype=torch.int32, device=dev)
        self.pool = self.k_pool = self.v_pool = None
        if kv_bits == 4:
            self.pool = paged.q4_pool(n_pages, page_rows, m.KV, m.D, layers=len(m.layers), device=dev)
        else:
            self.k_pool = torch.zeros((len(m.layers), n_pages, page_rows, m.KV, m.D), dtype=dtype, device=dev)
            self.v_pool = torch.zeros_like(self.k_pool)
        self.table = torch.zeros((requests, -(-max_len // page_rows)), **i32)
        self.ring = torch.arange(n_pages, **i32)
        self.ring_state = torch.tensor([0, n_pages], **i32)
        self.lens = torch.zeros(requests, **i32)
        self.held = torch.zeros(requests, **i32)
        self._rows = [0] * requests  # lens, as the host knows them
        self.cos, self.sin = device.rope_tables(max_len, m.D, m.rope_base, device=dev)
        self.w = [dict(qkv=_dequant(ly["wqkv"], dtype), wo=_dequant(ly["wo"], dtype),
                       gu=ChunkPrefill._gate_up(_dequant(ly["wgu"], dtype), m.F),
                       down=_dequant(ly["w_down"], dtype)) for ly in m.layers]

    def _check(self, sequences):
        """Refuse what the kernels would leave out: a count of requests that is not
        this step's, tokens outside the vocabulary, rows past max_len."""
        if len(sequences) != self.B:
            raise _lib.B2AShapeError(_lib.ERR_SHAPE, f"{len(sequences)} requests for {self.B}")
        for b, ids in enumerate(sequences):
            if self._rows[b] + len(ids) > self.max_len:
                raise _lib.B2AShapeError(
                    _lib.ERR_SHAPE, f"request {b}: {self._rows[b]} cached rows and {len(ids)} tokens "
                    f"exceed max_len {self.max_len}")
            if not all(0 <= t < self.m.V for t in ids):
                raise _lib.B2AShapeError(_lib.ERR_ARG, f"request {b}: a token outside [0, {self.m.V})")

    def _norm(self, x, w):
        h = torch.empty(x.shape, dtype=self.dt, device=x.device)
        _lib.check(_lib.load().b2a_rmsnorm_rows(
            x.data_ptr(), self.m.E, w.data_ptr(), self.m.eps, h.data_ptr(), self.m.E,
            device._code(self.dt), x.shape[0], self.m.E, device._stream(None)))
        return h

    def _forward(self, add, tokens, parents):
        """The nodes' logits (n, V) f32.  add: nodes per request; tokens and
        parents int32 device tensors of all nodes (parents None: chains)."""
        m, n = self.m, tokens.numel()
        add_dev = torch.tensor(add, dtype=torch.int32, device=m.device)
        plan = paged.page_plan(self.lens, add_dev, self.held, self.table, self.ring, self.ring_state,
                               page_rows=self.page_rows, max_tokens=n, parents=parents)
        if int(plan.slots.min()) < 0:  # the pages taken so far stay with the requests they went to
            self.held, self.ring_state = plan.held, plan.ring_state
            raise _lib.B2AError(_lib.ERR_WORKSPACE, "the cache has no pages left for a request")
        self.held, self.ring_state = plan.held, plan.ring_state
        x = torch.empty((n, m.E), dtype=torch.float32, device=m.device)
        _lib.check(_lib.load().b2a_q8_embed(
            m.tok_embd.codes.data_ptr(), m.tok_embd.scales.data_ptr(), m.V, m.E, tokens.data_ptr(),
            n, x.data_ptr(), device._stream(None)))
        nodes = max(add)
        for li, (ly, w) in enumerate(zip(m.layers, self.w)):
            qkv = device.gemm(self._norm(x, ly["attn_norm"]), w["qkv"]).view(n, m.H + 2 * m.KV, m.D)
            rows = (qkv[:, :m.H], qkv[:, m.H:m.H + m.KV], qkv[:, m.H + m.KV:], plan.positions,
                    plan.slots, self.cos, self.sin)
            turn = dict(style=m.rope_style, q_norm=ly.get("q_norm"), k_norm=ly.get("k_norm"), eps=m.eps)
            tree = dict(table=self.table, max_nodes=nodes, max_len=self.max_len)
            if self.pool is not None:
                q = paged.rope_append_q4(*rows, pool=self.pool[li], **turn,
                                         q_out=torch.empty((n, m.H, m.D), dtype=self.dt, device=m.device))
                att = paged.tree_decode_q4(q, self.pool[li], self.lens, plan.cu, parents, **tree)
            else:
                kp, vp = self.k_pool[li], self.v_pool[li]
                q = paged.rope_append(*rows, k_pool=kp, v_pool=vp, **turn)
                att = paged.tree_decode(q, kp, vp, self.lens, plan.cu, parents, **tree)
            device.gemm(att.view(n, m.H * m.D), w["wo"], out=x, c_in=x)
            act = torch.empty((n, m.F), dtype=self.dt, device=m.device)
            device.gemm(self._norm(x, ly["ffn_norm"]), w["gu"], out=act, epilogue=device.GEMM_SWIGLU)
            device.gemm(act, w["down"], out=x, c_in=x)
        return device.gemm_q8(self._norm(x, m.out_norm), m.output), plan

    def prefill(self, prompts):
        """Append prompts (a list of ids per request, empty: none) to the
        requests; returns each request's pick after its last token (-1: no
        prompt) as a list.  Where pages run out between two chunks of
        paged.MAX_NODES, those before are in the cache (`lens` says how far each
        request came)."""
        self._check(prompts)
        last = [-1] * self.B
        done = [0] * self.B
        while any(done[b] < len(p) for b, p in enumerate(prompts)):
            chunk = [p[done[b]:done[b] + paged.MAX_NODES] for b, p in enumerate(prompts)]
            add = [len(c) for c in chunk]
            tokens = torch.tensor(sum(chunk, []), dtype=torch.int32, device=self.m.device)
            logits, plan = self._forward(add, tokens, None)
            _, picks = paged.constrain_logits(logits, plan.cu, None, None, max_nodes=max(add), out=logits)
            self.lens = self.lens + torch.tensor(add, dtype=torch.int32, device=self.m.device)
            self._rows = [r + a for r, a in zip(self._rows, add)]
            picks, at = picks.tolist(), 0
            for b, c in enumerate(chunk):
                at += len(c)
                done[b] += len(c)
                if c and done[b] == len(prompts[b]):
                    last[b] = picks[at - 1]
        return last

    def verify(self, trees, *, uniforms=None, draws=None, temperature=None, draft=None, **limits):
        """One step.  trees: per request (tokens, parents) with the request's
        last token (not yet in the cache) as node 0, or None.  limits: the
        history, penalty, bias and mask arguments of paged.constrain_logits.
        Greedy unless draws (requests,) f32 and uniforms f32 of all nodes are
        given: then tokens are sampled with these numbers from [0, 1), with
        temperature and the drafts' own rows as paged.verify_picks takes them.
        Returns per request the tokens that are new: the accepted drafts and the
        model's own next token (None without a tree)."""
        if (uniforms is None) != (draws is None) or (draws is None and (temperature is not None or draft is not None)):
            raise _lib.B2AShapeError(_lib.ERR_ARG, "sampling needs uniforms and draws")
        self._check([() if t is None else t[0] for t in trees])
        for b, t in enumerate(trees):
            if t is None:
                continue
            if not 0 < len(t[0]) <= paged.MAX_NODES or len(t[1]) != len(t[0]):
                raise _lib.B2AShapeError(
                    _lib.ERR_SHAPE, f"request {b}: a tree needs 1 to {paged.MAX_NODES} tokens, each with a parent")
            if not all(-1 <= p < i for i, p in enumerate(t[1])):
                raise _lib.B2AShapeError(_lib.ERR_ARG, f"request {b}: a parent that is not an earlier node")
        if all(t is None for t in trees):
            return [None] * self.B
        add = [0 if t is None else len(t[0]) for t in trees]
        flat = [x for t in trees if t is not None for x in t[0]]
        par = [x for t in trees if t is not None for x in t[1]]
        if draws is not None:  # (refused before the step takes pages)
            for name, t, n in (("uniforms", uniforms, len(flat)), ("draws", draws, self.B),
                               ("temperature", temperature, self.B)):
                paged._f32(name, t, n)
            if draft is not None and (draft.dtype is not torch.float32 or not draft.is_cuda or
                                      draft.shape != (len(flat), self.m.V) or draft.stride(1) != 1 or
                                      (len(flat) > 1 and draft.stride(0) < self.m.V)):
                raise _lib.B2AShapeError(_lib.ERR_SHAPE, "draft must be a CUDA f32 tensor, a row per node")
        dev = self.m.device
        tokens = torch.tensor(flat, dtype=torch.int32, device=dev)
        parents = torch.tensor(par, dtype=torch.int32, device=dev)
        logits, plan = self._forward(add, tokens, parents)
        self.logits = logits
        # (sampled without limits: nothing to do to the logits, and no use for all rows' greedy
        # picks; verify_picks reads the rows on the paths alone)
        if draws is None or any(x is not None for x in limits.values()):
            _, self.picks = paged.constrain_logits(
                logits, plan.cu, parents, tokens, max_nodes=max(add), out=logits, **limits)
        if draws is not None:
            self.picks = paged.verify_picks(self.logits, plan.cu, parents, tokens, uniforms, draws,
                                            max_nodes=max(add), temperature=temperature, draft=draft)
        commit = dict(table=self.table, max_nodes=max(add), max_len=self.max_len)
        if self.pool is not None:
            c = paged.tree_commit_q4(self.picks, tokens, parents, plan.cu, self.lens, self.pool, **commit)
        else:
            c = paged.tree_commit(self.picks, tokens, parents, plan.cu, self.lens, self.k_pool,
                                  self.v_pool, **commit)
        self.lens = c.lens
        path, accepted, nxt = c.path.tolist(), c.accepted.tolist(), c.next_token.tolist()
        self._rows = [r + a for r, a in zip(self._rows, accepted)]
        return [None if t is None else [t[0][i] for i in path[b][1:accepted[b]]] + [nxt[b]]
                for b, t in enumerate(trees)]

    def end(self, requests):
        """Give the pages of finished requests back."""
        add = [-1 if b in requests else 0 for b in range(self.B)]
        dev = self.m.device
        plan = paged.page_plan(self.lens, torch.tensor(add, dtype=torch.int32, device=dev), self.held,
                               self.table, self.ring, self.ring_state, page_rows=self.page_rows,
                               max_tokens=0)
        self.held, self.ring_state = plan.held, plan.ring_state
        gone = torch.tensor([b in requests for b in range(self.B)], device=dev)
        self.lens = torch.where(gone, 0, self.lens).int()
        self._rows = [0 if b in requests else r for b, r in enumerate(self._rows)]
