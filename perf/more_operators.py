"""Measured cases of the operators that serve models with normed heads from a 4-bit
paged KV cache and verify drafted tokens by sampling.

  norm    RMSNorm of each head of q and k with the rotation in the same pass, the K/V
          rows stored at their slots of a 16-bit pool
  append  the same into a 4-bit pool (blocks of 32 values with a scale), and the rows as
          the pool holds them
  tree    the drafted tokens (the nodes of a tree per request; one node is an ordinary
          decode token) against a request's rows in a 4-bit pool
  verify  which drafted tokens stand and what follows them, from the model's
          probabilities and given random numbers

`run` computes each operator in its plain form (elementary torch operations in 32
bits, rounded once at the end; 64 where a number decides something), or, where `own` is
true, through this package's entry points.  `exact` gives the floating outputs from the
definitions in 64 bits.

A 4-bit block is 32 values of one row: d = m / -8 with m the value of largest magnitude
(the negative one of two), rounded to 8 significant bits and kept as f16; value i is
d * (code - 8) with code = floor(x / d + 8.5) within 0 .. 15.

A 4-bit pool is uint8 (pages, KV heads, granules, 18 D): a granule holds 16 consecutive
rows of one head, 8 D bytes of K codes, 8 D of V codes, then the f16 scales of K and of V
as [row][block].  Codes come in 32-bit words of 8 consecutive dims: dim 2i in bits 4i ..
4i + 3, dim 2i + 1 in bits 4i + 16 .. 4i + 19.  K words: [128 dims][row][word of its
block][block]; V words: [word of the row][row].
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 2.0 ** -20  # about the usual 1e-6, the same number in 32 and 64 bits


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the drafted tokens of 16 requests, f32 rows as a projection leaves them
        dict(name="norm_trees", op="norm", batch=16, len_lo=500, len_hi=32000, new_lo=8, new_hi=16,
             heads=32, kv_heads=8, head_dim=128, src="f32", dtype="bf16", page=64, style="neox"),
        # the rows of one long prompt, 16-bit projections
        dict(name="norm_prompt", op="norm", batch=1, len_lo=0, len_hi=0, new_lo=8191, new_hi=8191,
             heads=32, kv_heads=8, head_dim=128, src="bf16", dtype="bf16", page=64, style="neox"),
        # the same two into four bits: a step's drafts, and a prompt of odd length
        dict(name="append_trees", op="append", batch=16, len_lo=500, len_hi=32000, new_lo=8,
             new_hi=16, heads=32, kv_heads=8, head_dim=128, src="f32", dtype="f16", page=64,
             style="neox"),
        dict(name="append_prompt", op="append", batch=1, len_lo=0, len_hi=0, new_lo=8191,
             new_hi=8191, heads=32, kv_heads=8, head_dim=64, src="f16", dtype="f16", page=16,
             style="norm"),
        # one token of one short conversation: the smallest call, where latency counts
        dict(name="tree_single", op="tree", batch=1, len_lo=511, len_hi=511, new_lo=1, new_hi=1,
             heads=32, kv_heads=8, head_dim=64, dtype="f16", page=16),
        # a batch of ordinary conversations of any length, one token each
        dict(name="tree_ragged", op="tree", batch=64, len_lo=200, len_hi=7999, new_lo=1, new_hi=1,
             heads=32, kv_heads=8, head_dim=64, dtype="f16", page=16),
        # 16 long conversations, one token each: the cache is what is read
        dict(name="tree_long", op="tree", batch=16, len_lo=32760, len_hi=32760, new_lo=1,
             new_hi=1, heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=64),
        # the same conversations with eight drafted tokens each
        dict(name="tree_drafts", op="tree", batch=16, len_lo=32760, len_hi=32760, new_lo=8,
             new_hi=8, heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=64),
        # wide trees (up to 64 nodes x 8 heads a KV head) over ragged contexts: products
        dict(name="tree_wide", op="tree", batch=8, len_lo=9001, len_hi=16384, new_lo=33,
             new_hi=64, heads=64, kv_heads=8, head_dim=128, dtype="bf16", page=128),
        # one request's drafts, as a single-stream server verifies them
        dict(name="verify_single", op="verify", batch=1, new_lo=4, new_hi=4, vocab=128256,
             src="f32", draft=False),
        # the trees of 64 requests
        dict(name="verify_trees", op="verify", batch=64, new_lo=1, new_hi=31, vocab=128256,
             src="f32", draft=False),
        # drafts of a small model, whose distributions are known
        dict(name="verify_drafts", op="verify", batch=24, new_lo=5, new_hi=9, vocab=128256,
             src="f32", draft=True),
    ]


def draw(rng):
    def log(lo, hi):  # whole numbers spread over their logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def span(lo, hi):
        a, b = sorted((log(lo, hi), log(lo, hi)))
        return a, b

    top = {op: max(_cost(c) for c in listed() if c["op"] == op)
           for op in ("norm", "append", "tree", "verify")}
    while True:
        op = rng.choice(("norm", "append", "tree", "tree", "verify"))
        c = dict(op=op, batch=log(1, 64))
        heads, kv = rng.choice(((32, 8), (64, 8), (16, 2), (8, 8), (12, 4)))
        dim = rng.choice((64, 128, 256))
        page = rng.choice((16, 32, 64, 128))
        if op in ("norm", "append"):
            c["len_lo"], c["len_hi"] = span(1, 30000)
            c["new_lo"], c["new_hi"] = span(1, 8192 if c["batch"] < 4 else 64)
            c.update(heads=heads, kv_heads=kv, head_dim=dim, src=rng.choice(("f32", "f16", "bf16")),
                     dtype=rng.choice(("f32", "f16", "bf16") if op == "norm" else ("f16", "bf16")),
                     page=page, style=rng.choice(("norm", "neox")))
        elif op == "tree":
            c["len_lo"], c["len_hi"] = span(1, 32760)
            c["new_lo"], c["new_hi"] = span(1, 128)
            c.update(heads=heads, kv_heads=kv, head_dim=dim, dtype=rng.choice(("bf16", "f16")),
                     page=page)
        else:
            c["new_lo"], c["new_hi"] = span(1, 128)
            c["vocab"] = log(1000, 160000)
            c.update(src=rng.choice(("f32", "f32", "f16", "bf16")), draft=rng.random() < 0.4)
        if _cost(c) <= top[op]:
            return c


def _cost(case):
    """What keeps a drawn case below the largest listed one of its kind: the sizes of
    the plain form's largest intermediates, which grow with every size of the case."""
    B, n = case["batch"], case.get("new_hi", 1)
    if case["op"] in ("norm", "append"):
        rows = sum(_pages(a + b, case["page"]) for a, b in zip(_spread(case, "len"), _spread(case, "new")))
        # (a pool is written out whole, so long contexts count too)
        return (sum(_spread(case, "new")) * (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
                + rows * case["page"] * case["kv_heads"] * case["head_dim"] // 16)
    if case["op"] == "tree":
        rows = case["len_hi"] + n
        flops = 4 * B * n * case["heads"] * case["head_dim"] * rows
        return max(4 * B * rows * case["kv_heads"] * case["head_dim"], flops // 128,
                   4 * B * case["heads"] * n * rows)
    return sum(_spread(case, "new")) * case["vocab"] * (4 if case["draft"] else 1)


def _pages(rows, page):
    return -(-rows // page)


def _spread(case, what):
    """The batch's lengths (or node counts), evenly over [lo, hi]; prepare() deals them
    to the requests in an order of the seed's."""
    lo, hi, n = case[what + "_lo"], case[what + "_hi"], case["batch"]
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def work(case):
    op = case["op"]
    new = _spread(case, "new")
    N = sum(new)
    if op in ("norm", "append"):
        H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
        kept = 2 * KV * D * (BYTES[case["dtype"]] if op == "norm" else 9 / 16)
        row = (H + 2 * KV) * D * BYTES[case["src"]] + H * D * BYTES[case["dtype"]] + kept
        return {"bytes": int(N * (row + 8 + 4 * D)), "flops": 7 * N * (H + KV) * D}
    if op == "tree":
        H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
        lens = _spread(case, "len")
        rows = sum(a + b for a, b in zip(lens, new))
        pairs = sum(b * (a + 1) for a, b in zip(lens, new))  # each node: the prefix and itself
        return {"bytes": rows * KV * D * 9 // 8 + 2 * N * H * D * 2, "flops": 4 * pairs * H * D}
    # verify: with these drafts a path has 2.4 nodes on average, whatever the tree's size,
    # and only their rows decide anything
    path = min(2.4, N / case["batch"]) * case["batch"]
    row = case["vocab"] * (BYTES[case["src"]] + (4 if case["draft"] else 0))
    return {"bytes": int(path * row) + 16 * N, "flops": int(4 * path * case["vocab"])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _randn(shape, dtype, gen):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tree(n, rs):
    """Parents of a draft tree: node 0 is the root, the others hang near the front of
    what is there, as a beam's drafts do."""
    p = [-1]
    for i in range(1, n):
        p.append(int(rs.randint(max(0, i - 6), i)))
    return p[:n]


def _shifts(device):
    return torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=device)


def _filled_pool(shape, gen):
    """A 4-bit pool (pages, rows, KV, D) of random rows; some channels are larger than
    others, as keys have them."""
    P, R, KV, D = shape
    pool = torch.empty((P, KV, R // 16, 18 * D), dtype=torch.uint8, device="cuda")
    size = (0.4 * _randn((2, KV, 1, 1, D), torch.float32, gen)).exp()
    step = max(1, (1 << 26) // (R * KV * D))
    for lo in range(0, P, step):
        n = min(step, P - lo)
        parts, scales = [], []
        for s in (0, 1):
            x = _randn((n, KV, R // 16, 16, D), torch.float32, gen) * size[s]
            code, d = _to_codes(x)
            c = code.int()
            if s == 0:
                nb = min(4, D // 32)
                c = c.view(n, KV, R // 16, 16, -1, nb, 4, 8).permute(0, 1, 2, 4, 3, 6, 5, 7)
            else:
                c = c.view(n, KV, R // 16, 16, D // 8, 8).transpose(3, 4)
            word = (c << _shifts("cuda")).sum(-1).to(torch.int32)
            parts.append(word.reshape(n, KV, R // 16, 2 * D).view(torch.uint8))
            scales.append(d.reshape(n, KV, R // 16, D // 2).view(torch.uint8))
        pool[lo:lo + n] = torch.cat(parts + scales, -1)
    return pool


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator("cuda").manual_seed(seed)
    op, B = case["op"], case["batch"]
    order = rs.permutation(B)
    new = [_spread(case, "new")[i] for i in order]
    N = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s = {"case": dict(case), "cu": _ints(cu), "max_nodes": max(new)}
    if op in ("tree", "verify"):
        trees = [_tree(n, rs) for n in new]
        s["parents"] = _ints(sum(trees, []))
    if op == "verify":
        return _prepare_verify(case, s, trees, cu, rs, gen)
    lens = [_spread(case, "len")[i] for i in order]
    s["lens"] = _ints(lens)
    page = case["page"]
    H, KV, D, dt = case["heads"], case["kv_heads"], case["head_dim"], TYPES[case["dtype"]]
    s["max_len"] = max(a + b for a, b in zip(lens, new))
    # pages dealt out in no order, as a pool looks after a while, with a few to spare
    counts = [_pages(a + b, page) for a, b in zip(lens, new)]
    total = sum(counts) + 3
    perm = rs.permutation(total).astype(np.int32)
    table = np.zeros((B, max(counts) + 1), np.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    s["table"] = torch.from_numpy(table).cuda()
    if op == "norm":
        s["k_pool"] = _randn((total, page, KV, D), dt, gen)
        s["v_pool"] = _randn((total, page, KV, D), dt, gen)
    else:
        s["pool"] = _filled_pool((total, page, KV, D), gen)
    if op == "tree":
        s["q"] = _randn((N, H, D), dt, gen)
        return s
    # one packed projection row per token: q, k and v beside each other
    qkv = _randn((N, H + 2 * KV, D), TYPES[case["src"]], gen)
    s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    s["q_norm"] = 1 + 0.2 * _randn((D,), torch.float32, gen)
    s["k_norm"] = 1 + 0.2 * _randn((D,), torch.float32, gen)
    theta = torch.outer(torch.arange(s["max_len"] + 1, device="cuda", dtype=torch.float64),
                        1e6 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
    s["cos"], s["sin"] = theta.cos().float(), theta.sin().float()
    seqs = np.repeat(np.arange(B), new)
    row = np.concatenate([np.arange(a, a + n) for a, n in zip(lens, new)])
    slots = table[seqs, row // page] * page + row % page
    if N > 8:
        slots[rs.randint(N)] = -1  # a padding row: rotated, stored nowhere
    s["positions"], s["slots"] = _ints(row.tolist()), _ints(slots.tolist())
    s["q_out"] = torch.empty((N, H, D), dtype=dt, device="cuda")
    return s


def _prepare_verify(case, s, trees, cu, rs, gen):
    """Rows in which a few tokens stand out, as a language model's do; drafts are each
    row's likeliest tokens, or come from a draft model that is near the target."""
    V, B, N = case["vocab"], case["batch"], cu[-1]
    x = _randn((N, V), torch.float32, gen) * 2
    likely = torch.randint(0, V, (N, 24), device="cuda", generator=gen)
    x.scatter_add_(1, likely, 6 + 8 * torch.rand((N, 24), device="cuda", generator=gen))
    s["logits"] = x.to(TYPES[case["src"]])
    s["temperature"] = torch.tensor(rs.choice([0.0, 0.7, 0.8, 1.0, 1.2], B), dtype=torch.float32,
                                    device="cuda")
    s["draft"] = None
    best = x.topk(8, 1).indices.cpu().numpy()
    if case["draft"]:
        z = x * 0.9 + 0.7 * _randn((N, V), torch.float32, gen)
        s["draft"] = torch.softmax(z, 1)
        best = torch.multinomial(s["draft"], 8, True, generator=gen).cpu().numpy()
    tokens = rs.randint(0, V, N)
    for b, tree in enumerate(trees):
        kids = {}
        for i in range(1, len(tree)):
            k = kids[tree[i]] = kids.get(tree[i], -1) + 1
            if case["draft"] or rs.rand() < 0.9:
                tokens[cu[b] + i] = best[cu[b] + tree[i], k]
    s["tokens"] = _ints(tokens.tolist())
    s["uniforms"] = torch.rand(N, device="cuda", generator=gen)
    s["draws"] = torch.rand(B, device="cuda", generator=gen)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_norm(s):
    from alpacca_open_sourced_by_jt_b200 import paged
    q = paged.rope_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["cos"], s["sin"],
                          k_pool=s["k_pool"], v_pool=s["v_pool"], style=s["case"]["style"],
                          q_out=s["q_out"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _own_append(s):
    from alpacca_open_sourced_by_jt_b200 import paged
    q = paged.rope_append_q4(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["cos"], s["sin"],
                             pool=s["pool"], style=s["case"]["style"], q_out=s["q_out"],
                             q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    k, v = paged.q4_rows(s["pool"], s["slots"], dtype=q.dtype)
    return {"q": q, "k": k, "v": v}


def _own_tree(s):
    from alpacca_open_sourced_by_jt_b200 import paged
    return paged.tree_decode_q4(s["q"], s["pool"], s["lens"], s["cu"], s["parents"],
                                table=s["table"], max_nodes=s["max_nodes"], max_len=s["max_len"])


def _own_verify(s):
    from alpacca_open_sourced_by_jt_b200 import paged
    return paged.verify_picks(s["logits"], s["cu"], s["parents"], s["tokens"], s["uniforms"],
                              s["draws"], max_nodes=s["max_nodes"], temperature=s["temperature"],
                              draft=s["draft"])


_OWN = {"norm": _own_norm, "append": _own_append, "tree": _own_tree, "verify": _own_verify}


# ---- plain forms ----------------------------------------------------------

def _owner(cu, n):
    """For rows 0..n-1: their request and their index in it."""
    t = torch.arange(n, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=cu.numel() - 2)
    return seq, t - cu[seq]


def _ancestry(parents, cu, seq, idx, wide):
    """(rows, wide) truth values: node j of the row's request is the row's node or one
    of its ancestors.  Each round follows the known ancestors' own, twice as far."""
    j = torch.arange(wide, device=parents.device)
    base = cu[seq]
    up = parents.long()
    sees = j[None, :] == idx[:, None]
    for _ in range(max(1, math.ceil(math.log2(wide + 1)))):
        has = up >= 0
        at = torch.where(has, base + up, 0)
        sees = sees | (sees[at] & has[:, None])
        up = torch.where(has, up[at], -1)
    return sees


def _to_codes(x):
    """(codes, scales) of f32 rows, a scale per 32 values."""
    b = x.unflatten(-1, (-1, 32))
    hi, lo = b.amax(-1), b.amin(-1)
    m = torch.where(hi > -lo, hi, lo)
    d = (m / -8).bfloat16().float().clamp(-8160, 8160).half()
    by = torch.where(d == 0, torch.inf, d.float())[..., None]
    return (b / by + 8.5).floor().clamp(0, 15).flatten(-2), d


def _values(granules):
    """K and V rows (..., 16, D) in f32 of granules (..., 18 D) bytes."""
    D = granules.shape[-1] // 18
    lead = granules.shape[:-1]
    codes = granules[..., :16 * D].contiguous().view(torch.int32)
    scales = granules[..., 16 * D:].contiguous().view(torch.float16).float()
    nb = min(4, D // 32)
    k = (codes[..., :2 * D, None] >> _shifts(codes.device)) & 15
    k = k.view(*lead, -1, 16, 4, nb, 8).movedim(-5, -4).transpose(-3, -2)
    k = (k.reshape(*lead, 16, D // 32, 32).float() - 8) * scales[..., :D // 2].view(*lead, 16, -1, 1)
    v = (codes[..., 2 * D:, None] >> _shifts(codes.device)) & 15
    v = v.view(*lead, D // 8, 16, 8).transpose(-3, -2)
    v = (v.reshape(*lead, 16, D // 32, 32).float() - 8) * scales[..., D // 2:].view(*lead, 16, -1, 1)
    return k.flatten(-2), v.flatten(-2)


def _normed(x, w):
    # the sum and the number that it decides in 64 bits: a code next to a border hangs on it
    x = x.float()
    mean = (x.double().square().sum(-1, keepdim=True) / x.shape[-1] + EPS).float()
    return x * (1.0 / mean.sqrt()) * w


def _turn(x, cos, sin, style):
    if style == "norm":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_heads(s):
    style, pos = s["case"]["style"], s["positions"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _turn(_normed(s["q"], s["q_norm"]), cos, sin, style)
    return q.to(s["q_out"].dtype), _turn(_normed(s["k"], s["k_norm"]), cos, sin, style)


def _plain_norm(s):
    q, k = _plain_heads(s)
    slots = s["slots"].long()
    kept = slots >= 0
    KV, D = s["k"].shape[1:]
    at = slots[kept]
    s["k_pool"].view(-1, KV, D)[at] = k.to(s["k_pool"].dtype)[kept]
    s["v_pool"].view(-1, KV, D)[at] = s["v"].float().to(s["v_pool"].dtype)[kept]
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_append(s):
    q, k = _plain_heads(s)
    kept = (s["slots"] >= 0)[:, None, None]
    out = {"q": q}
    for name, x in (("k", k), ("v", s["v"].float())):
        code, d = _to_codes(x)
        x = ((code - 8).unflatten(-1, (-1, 32)) * d.float()[..., None]).flatten(-2)
        out[name] = torch.where(kept, x, 0.0).to(q.dtype)
    return out


def _plain_tree(s):
    q, lens, table, T = s["q"], s["lens"].long(), s["table"], s["max_nodes"]
    N, H, D = q.shape
    B, KV, L = lens.numel(), s["pool"].shape[1], s["max_len"]
    cu = s["cu"].long()
    seq, idx = _owner(cu, N)
    per = s["pool"].shape[2]  # granules of a page
    gran = torch.arange(-(-L // 16), device=q.device)
    at = s["pool"][table.long()[:, gran // per], :, gran % per]  # (B, granules, KV, bytes)
    k, v = _values(at)
    k, v = (x.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :L] for x in (k, v))
    row = torch.arange(L, device=q.device)
    there = row[None, :] < (lens + (cu[1:] - cu[:-1]))[:, None]
    # rows past a request's end hold anything: they count as zeros, with no weight
    v = torch.where(there[:, None, :, None], v, 0.0)
    qp = q.new_zeros((B, T, H, D), dtype=torch.float32)
    qp[seq, idx] = q.float()
    qp = qp.view(B, T, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, D)
    score = (qp @ k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    del k
    # node i of a request sees the rows before the tree, its ancestors and itself
    tree = row[None, :] - lens[:, None]
    sees = torch.zeros((B, T, T), dtype=torch.bool, device=q.device)
    sees[seq, idx] = _ancestry(s["parents"], cu, seq, idx, T)
    inside = sees.gather(2, tree.clamp(0, T - 1)[:, None, :].expand(B, T, L))
    seen = ((tree < 0)[:, None, :] | (inside & (tree < T)[:, None, :])) & there[:, None, :]
    score = score.view(B, KV, -1, T, L).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    score = (score - top).exp_()
    total = score.sum(-1, keepdim=True)
    out = score.view(B, KV, -1, L) @ v
    out = out.view(B, KV, -1, T, D) / total.clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, T, H, D)
    return out[seq, idx].to(q.dtype)


def _plain_verify(s):
    # weights, sums and the decisions that hang on them in 64 bits
    x = s["logits"].double()
    (N, V), B = x.shape, s["draws"].numel()
    cu = s["cu"].long()
    seq, idx = _owner(cu, N)
    tokens, parents, T = s["tokens"].long(), s["parents"].long(), s["max_nodes"]
    me = torch.arange(N, device=cu.device)
    child = parents >= 0
    up = torch.where(child, cu[seq] + parents, N)  # N: none
    top = x.amax(1, keepdim=True)
    ids = torch.arange(V, device=cu.device)
    best = torch.where(x == top, ids, V).amin(1)
    heat = s["temperature"].double()[seq][:, None]
    r = torch.where(heat > 0, ((x - top) / torch.where(heat > 0, heat, 1.0)).exp(),
                    (ids == best[:, None]).double())
    del x
    total = r.sum(1)
    # a node's children in turn, round k all nodes' k-th ones
    rank = ((up[:, None] == up[None, :]) & (me[None, :] < me[:, None])).sum(1)
    step = torch.full((N + 1,), N, dtype=torch.long, device=cu.device)
    rounds = int(torch.where(child, rank, -1).max()) + 1
    for k in range(rounds):
        c = torch.full((N + 1,), N, dtype=torch.long, device=cu.device)
        c[torch.where(child & (rank == k), up, N)] = me
        c = c[:N]
        has = (c < N) & (step[:N] == N)  # nodes that have a k-th child to look at
        at = torch.where(has, c, 0)
        tok = tokens[at]
        mine = r.gather(1, tok[:, None])[:, 0]
        u = s["uniforms"].double()[at]
        if s["draft"] is None:
            take = has & (u * total < mine)
            gone = has & ~take
            r.scatter_(1, tok[:, None], torch.where(gone, 0.0, mine)[:, None])
        else:
            q = s["draft"].gather(1, tok[:, None])[:, 0].double()
            take = has & (u * q * total < mine)
            gone = has & ~take
            rest = (r[gone] / total[gone, None] - s["draft"][gone].double()).clamp(min=0)
            r[gone] = rest.scatter(1, tok[gone, None], 0.0)
        total = torch.where(gone, r.sum(1), total)
        step[:N] = torch.where(take, at, step[:N])
    node = torch.where(cu[1:] > cu[:-1], cu[:-1], N)  # the root of each request
    picks = torch.full((N + 1,), -1, dtype=torch.int32, device=cu.device)
    last = node
    ext = torch.cat([tokens, tokens.new_full((1,), -1)]).int()
    for _ in range(T):
        last = torch.where(node < N, node, last)
        nxt = torch.where(node < N, step[node], N)
        picks[node] = torch.where(nxt < N, ext[nxt], picks[node])
        node = nxt
    there = last < N
    row = r[torch.where(there, last, 0)]
    cum = row.cumsum(1)
    goal = (s["draws"].double() * cum[:, -1])[:, None]
    drawn = torch.searchsorted(cum, goal, right=True)[:, 0].clamp(max=V - 1)
    picks[last] = torch.where(there, drawn.int(), -1)
    return picks[:N]


_PLAIN = {"norm": _plain_norm, "append": _plain_append, "tree": _plain_tree, "verify": _plain_verify}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers only
    s = prepare(case, seed)
    return _EXACT[case["op"]](s)


def _exact_heads(s, x, w):
    """Normed and turned heads, each pair as one complex number."""
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    pos = s["positions"].tolist()
    turn = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None]
    half = x.shape[-1] // 2
    if s["case"]["style"] == "norm":
        return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (half, 2)).contiguous()) * turn).flatten(-2)
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
    return torch.cat([z.real, z.imag], -1)


def _exact_norm(s):
    kept = [t for t, at in enumerate(s["slots"].tolist()) if at >= 0]
    at = s["slots"].long()[kept]
    k, v = s["k_pool"].double(), s["v_pool"].double()
    k.flatten(0, 1)[at] = _exact_heads(s, s["k"], s["k_norm"])[kept]
    v.flatten(0, 1)[at] = s["v"].double()[kept]
    return {"q": _exact_heads(s, s["q"], s["q_norm"]), "k_pool": k, "v_pool": v}


def _exact_append(s):
    out = {"q": _exact_heads(s, s["q"], s["q_norm"])}
    for name, x in (("k", _exact_heads(s, s["k"], s["k_norm"])), ("v", s["v"].double())):
        x = x.unflatten(-1, (-1, 32))
        far = x.abs().amax(-1, keepdim=True)
        d = torch.where((x == -far).any(-1, keepdim=True), -far, far) / -8
        part, power = torch.frexp(d)  # 8 significant bits
        d = torch.ldexp((part * 256).round() / 256, power).half().double()
        code = torch.clamp(torch.floor(x / torch.where(d == 0, 1.0, d) + 8.5), 0, 15)
        y = torch.where(d == 0, 0.0, d * (code - 8)).flatten(-2)
        y[(s["slots"] < 0).nonzero()[:, 0]] = 0
        out[name] = y
    return out


def _chain(parents, i):
    """Node i and its ancestors."""
    found = []
    while i >= 0:
        found.append(i)
        i = parents[i]
    return found


def _exact_rows(pool, pages):
    """K and V rows of one request's pages, (KV, rows, D) in 64 bits, dim by dim."""
    g = pool[pages.long()].transpose(0, 1).flatten(1, 2)  # (KV, granules, bytes)
    KV, G, D = g.shape[0], g.shape[1], g.shape[2] // 18
    word = g[..., :16 * D].contiguous().view(torch.int32).long() & 0xffffffff
    scale = g[..., 16 * D:].contiguous().view(torch.float16).double().view(KV, G, 2, 16, D // 32)
    nb = min(4, D // 32)
    r = torch.arange(16, device=g.device)
    out = torch.empty((2, KV, G, 16, D), dtype=torch.float64, device=g.device)
    for dim in range(D):
        block, w, i = dim // 32, dim % 32 // 8, dim % 8
        shift = 4 * (i // 2) + 16 * (i % 2)
        at_k = dim // 128 * 64 * nb + r * 4 * nb + w * nb + block % 4
        at_v = 2 * D + dim // 8 * 16 + r
        for which, at in ((0, at_k), (1, at_v)):
            out[which, ..., dim] = (((word[..., at] >> shift) & 15) - 8) * scale[:, :, which, :, block]
    return out.flatten(2, 3)


def _exact_tree(s):
    q = s["q"].double()
    H, D = q.shape[1:]
    KV, page = s["pool"].shape[1], 16 * s["pool"].shape[2]
    cu, lens, parents = s["cu"].tolist(), s["lens"].tolist(), s["parents"].tolist()
    out = torch.empty_like(q)
    for b, ln in enumerate(lens):
        n = cu[b + 1] - cu[b]
        k, v = _exact_rows(s["pool"], s["table"][b, :_pages(ln + n, page)])[:, :, :ln + n]
        blind = torch.ones((n, n), dtype=torch.bool)
        for i in range(n):
            blind[i, _chain(parents[cu[b]:cu[b + 1]], i)] = False
        blind = blind.cuda()
        for g in range(KV):
            heads = slice(g * (H // KV), (g + 1) * (H // KV))
            x = q[cu[b]:cu[b + 1], heads] @ k[g].T / math.sqrt(D)
            x[:, :, ln:].masked_fill_(blind[:, None, :], -math.inf)
            out[cu[b]:cu[b + 1], heads] = torch.softmax(x, -1) @ v[g]
    return out


_EXACT = {"norm": _exact_norm, "append": _exact_append, "tree": _exact_tree}
