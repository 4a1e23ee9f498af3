"""Measured cases of the operators that serve many requests from one paged KV
cache and verify trees of drafted tokens over it.

One serving step of such a loop is, per model layer or once per step:

  plan       block tables, slot map and positions of the step's tokens, built on
             the GPU from the requests' lengths (pages taken from and given back
             to a ring of free pages)
  append     RoPE of q and k, the K/V rows stored at their slots
  attention  the drafted tokens (the nodes of a tree per request; one node is an
             ordinary decode token) against the request's cached rows and their
             own ancestors
  logits     penalties for repeated tokens, logit biases and grammar masks on the
             rows of the LM head, and the row's greedy pick
  commit     the longest accepted path of each tree, its K/V rows moved to their
             final places in every layer

`run` computes each operator in its plain form (elementary torch operations in 32
bits, rounded once at the end), or, where `own` is true, through this package's
entry points.  `exact` gives the floating outputs from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decode step's bookkeeping: 64 requests, each with a small draft tree
        dict(name="plan_trees", op="plan", batch=64, len_lo=1000, len_hi=8192, new_lo=1,
             new_hi=16, page=64, tree=True, ending=3),
        # admission of a wave of prompts (short questions to long documents) while a
        # few requests end: about half a million slots over small pages
        dict(name="plan_prompts", op="plan", batch=251, len_lo=0, len_hi=900, new_lo=1,
             new_hi=4096, page=16, tree=False, ending=20),
        # the drafted tokens of 16 requests, f32 rows as a projection leaves them
        dict(name="append_trees", op="append", batch=16, len_lo=500, len_hi=32000, new_lo=8,
             new_hi=16, heads=32, kv_heads=8, head_dim=128, src="f32", dtype="bf16", page=64,
             style="norm"),
        # the rows of one long prompt, 16-bit projections, split-halves rotation
        dict(name="append_prompt", op="append", batch=1, len_lo=0, len_hi=0, new_lo=8191,
             new_hi=8191, heads=32, kv_heads=8, head_dim=64, src="f16", dtype="f16", page=16,
             style="neox"),
        # one token of one short conversation: the smallest call, where latency counts
        dict(name="tree_single", op="tree", batch=1, len_lo=511, len_hi=511, new_lo=1, new_hi=1,
             heads=32, kv_heads=8, head_dim=64, dtype="f16", page=16),
        # 16 long conversations, eight drafted tokens each: the cache is what is read
        dict(name="tree_long", op="tree", batch=16, len_lo=32760, len_hi=32760, new_lo=8,
             new_hi=8, heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=64),
        # wide trees (up to 64 nodes x 8 heads a KV head) over ragged contexts: products
        dict(name="tree_wide", op="tree", batch=8, len_lo=9001, len_hi=16384, new_lo=33,
             new_hi=64, heads=64, kv_heads=8, head_dim=128, dtype="bf16", page=128),
        # an f32 cache in one block per sequence, odd lengths
        dict(name="tree_f32", op="tree", batch=3, len_lo=77, len_hi=2049, new_lo=1, new_hi=12,
             heads=32, kv_heads=8, head_dim=128, dtype="f32", page=0),
        # one row, as a single-stream decode makes it
        dict(name="logits_single", op="logits", batch=1, new_lo=1, new_hi=1, vocab=128256,
             hist_lo=700, hist_hi=700, biases=8, mask=True, src="f32", dst="f32"),
        # every node of 64 requests' trees, long histories
        dict(name="logits_trees", op="logits", batch=64, new_lo=1, new_hi=31, vocab=128256,
             hist_lo=10, hist_hi=8192, biases=32, mask=True, src="f32", dst="f32"),
        # one request of a 16-layer model, 64-wide heads
        dict(name="commit_single", op="commit", batch=1, len_lo=4000, len_hi=4000, new_lo=16,
             new_hi=16, layers=16, kv_heads=8, head_dim=64, dtype="f16", page=16),
        # 64 requests, 128-wide heads, trees of 8 to 32 nodes
        dict(name="commit_trees", op="commit", batch=64, len_lo=100, len_hi=1000, new_lo=8,
             new_hi=32, layers=16, kv_heads=8, head_dim=128, dtype="bf16", page=64),
    ]


def draw(rng):
    def log(lo, hi):  # whole numbers spread over their logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def span(lo, hi):
        a, b = sorted((log(lo, hi), log(lo, hi)))
        return a, b

    top = {op: max(_cost(c) for c in listed() if c["op"] == op)
           for op in ("plan", "append", "tree", "logits", "commit")}
    while True:
        op = rng.choice(("plan", "append", "tree", "tree", "logits", "commit"))
        c = dict(op=op, batch=log(1, 256 if op == "plan" else 64))
        heads, kv = rng.choice(((32, 8), (64, 8), (16, 2), (8, 8), (12, 4)))
        dim = rng.choice((64, 128, 256))
        page = rng.choice((16, 32, 64, 128))
        if op == "plan":
            c["len_lo"], c["len_hi"] = span(1, 32768)
            c["tree"] = rng.random() < 0.5
            c["new_lo"], c["new_hi"] = span(1, 128 if c["tree"] else 4096)
            c["page"], c["ending"] = page, rng.randrange(0, c["batch"])
        elif op == "append":
            c["len_lo"], c["len_hi"] = span(1, 30000)
            c["new_lo"], c["new_hi"] = span(1, 8192 if c["batch"] < 4 else 64)
            c.update(heads=heads, kv_heads=kv, head_dim=dim, src=rng.choice(("f32", "f16", "bf16")),
                     dtype=rng.choice(("f32", "f16", "bf16")), page=page,
                     style=rng.choice(("norm", "neox")))
        elif op == "tree":
            c["len_lo"], c["len_hi"] = span(1, 32760)
            c["new_lo"], c["new_hi"] = span(1, 128)
            c.update(heads=heads, kv_heads=kv, head_dim=dim,
                     dtype=rng.choice(("bf16", "f16", "bf16", "f16", "f32")),
                     page=rng.choice((0, page, page)))
        elif op == "logits":
            c["new_lo"], c["new_hi"] = span(1, 128)
            c["vocab"] = log(1000, 160000)
            c["hist_lo"], c["hist_hi"] = span(1, 16384)
            c.update(biases=rng.randrange(0, 65), mask=rng.random() < 0.7,
                     src=rng.choice(("f32", "f16", "bf16")), dst=rng.choice(("f32", "f32", "bf16")))
        else:
            c["len_lo"], c["len_hi"] = span(1, 2000)
            c["new_lo"], c["new_hi"] = span(1, 128)
            c.update(layers=rng.randrange(1, 17), kv_heads=kv, head_dim=dim,
                     dtype=rng.choice(("f32", "f16", "bf16")), page=page)
        if _cost(c) <= top[op]:
            return c


def _cost(case):
    """What keeps a drawn case below the largest listed one of its kind: the sizes of
    the plain form's largest intermediates, which grow with every size of the case."""
    B, n = case["batch"], case.get("new_hi", 1)
    if case["op"] == "plan":
        return B * (n + (case["len_hi"] + n) // case["page"])
    if case["op"] == "append":
        return sum(_spread(case, "new")) * (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
    if case["op"] == "tree":
        rows = case["len_hi"] + n
        flops = 4 * B * n * case["heads"] * case["head_dim"] * rows
        if case["dtype"] == "f32":  # 32-bit products have no tensor cores
            flops *= 16
        return max(4 * B * rows * case["kv_heads"] * case["head_dim"], flops // 128,
                   4 * B * case["heads"] * n * rows)
    if case["op"] == "logits":
        return sum(_spread(case, "new")) * case["vocab"]
    rows = sum(_pages(ln + k, case["page"]) for ln, k in zip(_spread(case, "len"), _spread(case, "new")))
    return rows * case["page"] * case["layers"] * case["kv_heads"] * case["head_dim"]


def _pages(rows, page):
    return -(-rows // page)


def _spread(case, what):
    """The batch's lengths (or node counts, or history lengths), evenly over
    [lo, hi]; prepare() deals them to the requests in an order of the seed's."""
    lo, hi, n = case[what + "_lo"], case[what + "_hi"], case["batch"]
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def work(case):
    op = case["op"]
    new = _spread(case, "new")
    N = sum(new)
    if op == "plan":
        # lengths, counts and held pages in; tokens' request, position and slot out; the
        # new pages' table entries and the pages that come back
        ends = case["ending"]
        lens = _spread(case, "len")
        taken = sum(_pages(a + b, case["page"]) - _pages(a, case["page"])
                    for a, b in zip(lens[ends:], new[ends:]))
        back = sum(_pages(a, case["page"]) for a in lens[:ends])
        tokens = sum(new[ends:])
        return {"bytes": 4 * (6 * case["batch"] + 3 * tokens + tokens * case["tree"]
                              + 2 * taken + 2 * back), "flops": 3 * tokens}
    if op == "append":
        H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
        rows = N * (H + 2 * KV) * D
        return {"bytes": rows * (BYTES[case["src"]] + BYTES[case["dtype"]]) + N * (8 + 4 * D),
                "flops": 3 * N * (H + KV) * D}
    if op == "tree":
        H, KV, D, es = case["heads"], case["kv_heads"], case["head_dim"], BYTES[case["dtype"]]
        lens = _spread(case, "len")
        rows = sum(a + b for a, b in zip(lens, new))
        pairs = sum(b * (a + 1) for a, b in zip(lens, new))  # each node: the prefix and itself
        return {"bytes": 2 * rows * KV * D * es + 2 * N * H * D * es, "flops": 4 * pairs * H * D}
    if op == "logits":
        V = case["vocab"]
        hist = sum(_spread(case, "hist"))
        return {"bytes": N * V * (BYTES[case["src"]] + BYTES[case["dst"]])
                + (N * V // 8 if case["mask"] else 0) + 4 * hist + 8 * case["biases"] * case["batch"]
                + 4 * N, "flops": 4 * N * V}
    # commit: with these trees and picks a path has 2.5 nodes on average, whatever the
    # tree's size, and the rows of 1.2 of them move
    row = 2 * case["layers"] * case["kv_heads"] * case["head_dim"] * BYTES[case["dtype"]]
    return {"bytes": int(2.4 * case["batch"] * row) + 16 * N, "flops": 4 * N}


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


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator("cuda").manual_seed(seed)
    op, B = case["op"], case["batch"]
    order = rs.permutation(B)
    new = [_spread(case, "new")[i] for i in order]
    s = {"case": dict(case)}
    if op == "plan":
        return _prepare_plan(case, s, rs, order)
    N = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s["cu"] = _ints(cu)
    s["max_nodes"] = max(new)
    if op in ("tree", "logits", "commit"):
        trees = [_tree(n, rs) for n in new]
        s["parents"] = _ints(sum(trees, []))
    if op == "logits":
        return _prepare_logits(case, s, rs, gen, new, order)
    lens = [_spread(case, "len")[i] for i in order]
    s["lens"] = _ints(lens)
    page = case["page"]
    KV, D, dt = case["kv_heads"], case["head_dim"], TYPES[case["dtype"]]
    layers = case.get("layers", 1)
    s["max_len"] = max(a + b for a, b in zip(lens, new))
    if page:
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
        shape = (total, page, KV, D)
    else:
        s["table"] = None
        shape = (B, s["max_len"] + 5, KV, D)
    if op == "commit":
        shape = (layers,) + shape
    s["k_pool"], s["v_pool"] = _randn(shape, dt, gen), _randn(shape, dt, gen)
    if op == "tree":
        s["q"] = _randn((N, case["heads"], D), dt, gen)
    elif op == "append":
        src = TYPES[case["src"]]
        H = case["heads"]
        # one packed projection row per token: q, k and v beside each other
        qkv = _randn((N, H + 2 * KV, D), src, gen)
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        rows = s["max_len"] + 1
        theta = torch.outer(torch.arange(rows, device="cuda", dtype=torch.float64),
                            500000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
        s["cos"], s["sin"] = theta.cos().float(), theta.sin().float()
        seqs = np.repeat(np.arange(B), new)
        row = np.concatenate([np.arange(a, a + n) for a, n in zip(lens, new)])
        slots = table[seqs, row // page] * page + row % page
        if N > 8:
            slots[rs.randint(N)] = -1  # a padding row: rotated, stored nowhere
        s["positions"], s["slots"] = _ints(row.tolist()), _ints(slots.tolist())
        s["q_out"] = torch.empty((N, H, D), dtype=dt, device="cuda")
    else:
        # drafts and the model's picks: most nodes have a child that holds their pick
        tokens = rs.randint(0, 32000, N)
        picks = rs.randint(0, 32000, N)
        for b, tree in enumerate(trees):
            for i in range(1, len(tree)):
                if rs.rand() < 0.5:
                    picks[cu[b] + tree[i]] = tokens[cu[b] + i]
        s["tokens"], s["picks"] = _ints(tokens.tolist()), _ints(picks.tolist())
    return s


def _prepare_plan(case, s, rs, order):
    B, page = case["batch"], case["page"]
    lens, new = _spread(case, "len"), _spread(case, "new")
    new = [-1 if i < case["ending"] else n for i, n in enumerate(new)]
    lens, new = [lens[i] for i in order], [new[i] for i in order]
    held = [_pages(a, page) for a in lens]
    wide = max(_pages(a + max(n, 0), page) for a, n in zip(lens, new)) + 2
    need = sum(max(0, _pages(a + n, page) - h) for a, n, h in zip(lens, new, held) if n > 0)
    free = max(1, need - need // 50)  # nearly all requests find their pages
    total = sum(held) + free
    perm = rs.permutation(total).astype(np.int32)
    table = np.full((B, wide), -1, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = perm[at:at + h]
        at += h
    ring = np.zeros(total, np.int32)
    head = int(rs.randint(total))
    ring[(head + np.arange(free)) % total] = perm[at:]
    tokens = sum(max(n, 0) for n in new)
    s.update(lens=_ints(lens), new=_ints(new), held=_ints(held), table=torch.from_numpy(table).cuda(),
             ring=torch.from_numpy(ring).cuda(), ring_state=_ints([head, free]),
             max_tokens=tokens + 7, page=page, parents=None)
    if case["tree"]:
        # padded like the rows of the step's other buffers
        s["parents"] = _ints(sum((_tree(max(n, 0), rs) for n in new), []) + [-1] * 7)
    return s


def _prepare_logits(case, s, rs, gen, new, order):
    B, V, N = case["batch"], case["vocab"], sum(new)
    hist = [_spread(case, "hist")[i] for i in order]

    def words(n):  # few tokens are frequent, most are rare
        return np.minimum((V * rs.rand(n) ** 4).astype(np.int64), V - 1)

    s["logits"] = (_randn((N, V), torch.float32, gen) * 4).to(TYPES[case["src"]])
    s["tokens"] = _ints(words(N).tolist())
    s["hist"] = _ints(words(sum(hist)).tolist())
    s["hist_start"] = _ints(np.concatenate([[0], np.cumsum(hist)]).tolist())
    s["prompt_lens"] = _ints([int(h * rs.rand()) for h in hist])
    f32 = dict(dtype=torch.float32, device="cuda")
    s["repetition"] = torch.tensor(rs.choice([1.0, 1.1, 1.3], B), **f32)
    s["presence"] = torch.tensor(rs.choice([0.0, 0.4, 1.0], B), **f32)
    s["frequency"] = torch.tensor(rs.choice([0.0, 0.1, 0.5], B), **f32)
    n = min(case["biases"], V)
    s["bias_start"] = _ints([n * b for b in range(B + 1)])
    s["bias_ids"] = _ints(np.concatenate([rs.choice(V, n, replace=False) for _ in range(B)]).tolist()
                          if n else [0])
    s["bias"] = torch.tensor(rs.randn(max(n * B, 1)) * 5, **f32)
    s["mask"] = None
    if case["mask"]:
        # a third of the rows stand at a place of their grammar where few tokens may
        # follow, the others are free; a dead end now and then leaves a row nothing
        wide = (V + 31) // 32
        bits = torch.randint(-2 ** 31, 2 ** 31, (N, wide), device="cuda", generator=gen)
        for _ in range(2):
            bits &= torch.randint(-2 ** 31, 2 ** 31, (N, wide), device="cuda", generator=gen)
        free = torch.from_numpy(rs.rand(N, 1) >= 0.33).cuda()
        bits = torch.where(free, -1, bits)
        if N > 8:
            bits[rs.randint(N)] = 0
        s["mask"] = bits.to(torch.int32)
    s["out"] = torch.empty((N, V), dtype=TYPES[case["dst"]], device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_plan(s):
    from alpacca_open_sourced_by_jt_b200 import paged
    p = paged.page_plan(s["lens"], s["new"], s["held"], s["table"], s["ring"], s["ring_state"],
                        page_rows=s["page"], max_tokens=s["max_tokens"], parents=s["parents"])
    return {"table": s["table"], "ring": s["ring"], "held": p.held, "ring_state": p.ring_state,
            "cu": p.cu, "seq": p.seq, "positions": p.positions, "slots": p.slots}


def _own_append(s):
    from alpacca_open_sourced_by_jt_b200 import paged
    q = paged.rope_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["cos"], s["sin"],
                          k_pool=s["k_pool"], v_pool=s["v_pool"], style=s["case"]["style"],
                          q_out=s["q_out"])
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _own_tree(s):
    from alpacca_open_sourced_by_jt_b200 import paged
    return paged.tree_decode(s["q"], s["k_pool"], s["v_pool"], s["lens"], s["cu"], s["parents"],
                             table=s["table"], max_nodes=s["max_nodes"], max_len=s["max_len"])


def _own_logits(s):
    from alpacca_open_sourced_by_jt_b200 import paged
    out, picks = paged.constrain_logits(
        s["logits"], s["cu"], s["parents"], s["tokens"], max_nodes=s["max_nodes"], hist=s["hist"],
        hist_start=s["hist_start"], prompt_lens=s["prompt_lens"], repetition=s["repetition"],
        presence=s["presence"], frequency=s["frequency"], bias_start=s["bias_start"],
        bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"], out=s["out"])
    return {"logits": out, "picks": picks}


def _own_commit(s):
    from alpacca_open_sourced_by_jt_b200 import paged
    c = paged.tree_commit(s["picks"], s["tokens"], s["parents"], s["cu"], s["lens"], s["k_pool"],
                          s["v_pool"], table=s["table"], max_nodes=s["max_nodes"])
    return {"path": c.path, "accepted": c.accepted, "next": c.next_token, "lens": c.lens,
            "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


_OWN = {"plan": _own_plan, "append": _own_append, "tree": _own_tree, "logits": _own_logits,
        "commit": _own_commit}


# ---- plain forms ----------------------------------------------------------

def _owner(cu, n):
    """For rows 0..n-1: their request (clamped for rows past the last), their index in
    it, and whether they belong to one."""
    t = torch.arange(n, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    valid = t < cu[-1]
    seq = seq.clamp(max=cu.numel() - 2)
    return seq, t - cu[seq], valid


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


def _plain_plan(s):
    page, ring, table = s["page"], s["ring"], s["table"]
    lens, new, held = s["lens"].long(), s["new"].long(), s["held"].long()
    size, wide = ring.numel(), table.shape[1]
    head, count = s["ring_state"].long()
    ends = new < 0
    n = new.clamp(min=0)
    want = (lens + n + page - 1) // page
    fits = want <= wide
    need = torch.where(ends | ~fits, 0, (want - held).clamp(min=0))
    upto = need.cumsum(0)
    served = ~ends & fits & ((need == 0) | (upto <= count))
    got = torch.where(served, need, 0)
    taken = torch.where(served & (need > 0), upto, 0).amax()
    j = torch.arange(wide, device=ring.device)
    k = j[None, :] - held[:, None]
    fresh = (k >= 0) & (k < got[:, None])
    at = (head + (upto - need)[:, None] + k) % size
    table_new = torch.where(fresh, ring[at.clamp(min=0)], table)
    back = torch.where(ends, held, 0)
    at = (head + count + (back.cumsum(0) - back)[:, None] + j[None, :]) % size
    gives = j[None, :] < back[:, None]
    ring_new = torch.cat([ring, ring.new_zeros(1)])
    ring_new[torch.where(gives, at, size).reshape(-1)] = torch.where(gives, table, 0).reshape(-1)
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)])
    seq, idx, valid = _owner(cu, s["max_tokens"])
    row = lens[seq] + idx
    ok = valid & served[seq]
    slot = table_new[seq, (row // page).clamp(max=wide - 1)].long() * page + row % page
    if s["parents"] is None:
        depth = idx
    else:
        depth = _ancestry(s["parents"], cu, seq, idx, 128).sum(1) - 1
    return {"table": table_new, "ring": ring_new[:-1],
            "held": torch.where(ends, 0, held + got).int(),
            "ring_state": torch.stack([(head + taken) % size, count - taken + back.sum()]).int(),
            "cu": cu.int(), "seq": torch.where(valid, seq, -1).int(),
            "positions": torch.where(valid, lens[seq] + depth, 0).int(),
            "slots": torch.where(ok, slot, -1).int()}


def _turn(x, cos, sin, style):
    if style == "norm":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_append(s):
    style, slots = s["case"]["style"], s["slots"].long()
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    kept = slots >= 0
    KV, D = s["k"].shape[1:]
    at = slots[kept]
    s["k_pool"].view(-1, KV, D)[at] = _turn(s["k"].float(), cos, sin, style).to(s["k_pool"].dtype)[kept]
    s["v_pool"].view(-1, KV, D)[at] = s["v"].float().to(s["v_pool"].dtype)[kept]
    return {"q": _turn(s["q"].float(), cos, sin, style).to(s["k_pool"].dtype),
            "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_tree(s):
    q, lens, table, T = s["q"], s["lens"].long(), s["table"], s["max_nodes"]
    N, H, D = q.shape
    B, KV, L = lens.numel(), s["k_pool"].shape[-2], s["max_len"]
    cu = s["cu"].long()
    seq, idx, _ = _owner(cu, N)
    row = torch.arange(L, device=q.device)
    page = s["k_pool"].shape[1]
    if table is None:
        at = torch.arange(B, device=q.device)[:, None] * page + row[None, :]
    else:
        at = table.long()[:, row // page] * page + row % page
    rows = lens + (cu[1:] - cu[:-1])
    there = row[None, :] < rows[:, None]
    # rows past a request's end hold anything: they count as zeros, with no weight
    k = s["k_pool"].view(-1, KV, D)[at].float()
    v = torch.where(there[:, :, None, None], s["v_pool"].view(-1, KV, D)[at].float(), 0.0)
    qp = q.new_zeros((B, T, H, D), dtype=torch.float32)
    qp[seq, idx] = q.float()
    qp = qp.view(B, T, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, D)
    score = (qp @ k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(D))
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
    out = score.view(B, KV, -1, L) @ v.transpose(1, 2)
    out = out.view(B, KV, -1, T, D) / total.clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, T, H, D)
    return out[seq, idx].to(q.dtype)


def _plain_logits(s):
    V, (N, B) = s["logits"].shape[1], (s["logits"].shape[0], s["cu"].numel() - 1)
    cu = s["cu"].long()
    seq, idx, _ = _owner(cu, N)
    start = s["hist_start"].long()
    hseq, hidx, _ = _owner(start, s["hist"].numel())
    prompt = hidx < s["prompt_lens"].long()[hseq]
    word = hseq * V + s["hist"].long()
    count = torch.zeros(B * V, dtype=torch.int32, device=cu.device)
    count.index_add_(0, word, (~prompt).int())
    told = torch.zeros(B * V, dtype=torch.int32, device=cu.device)
    told.index_add_(0, word, prompt.int())
    bseq, _, has = _owner(s["bias_start"].long(), s["bias_ids"].numel())
    bias = torch.zeros(B * V, dtype=torch.float32, device=cu.device)
    bias.index_add_(0, bseq * V + s["bias_ids"].long(), torch.where(has, s["bias"], 0.0))
    # the drafted tokens on a row's path count as said
    T = s["max_nodes"]
    path = _ancestry(s["parents"], cu, seq, idx, T)
    at = (cu[seq][:, None] + torch.arange(T, device=cu.device)[None, :]).clamp(max=N - 1)
    c = count.view(B, V)[seq]
    c.scatter_add_(1, s["tokens"].long()[at], path.int())
    seen = (c > 0) | (told.view(B, V)[seq] > 0)
    x = s["logits"].float() + bias.view(B, V)[seq]
    rep = s["repetition"][seq][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][seq][:, None] * c.float()
    x = torch.where(c > 0, x - s["presence"][seq][:, None], x)
    if s["mask"] is not None:
        v = torch.arange(V, device=cu.device)
        allowed = ((s["mask"][:, v // 32] >> (v % 32).int()) & 1) != 0
        x = x.masked_fill(~allowed, -math.inf)
    top = x.amax(1, keepdim=True)
    ids = torch.arange(V, device=cu.device, dtype=torch.int32)
    pick = torch.where(x == top, ids[None, :], V).amin(1)
    pick = torch.where(top[:, 0] == -math.inf, -1, pick)
    return {"logits": x.to(s["out"].dtype), "picks": pick.int()}


def _plain_commit(s):
    cu, lens, T = s["cu"].long(), s["lens"].long(), s["max_nodes"]
    N, B = s["tokens"].numel(), s["lens"].numel()
    seq, idx, _ = _owner(cu, N)
    parents, tokens, picks = s["parents"].long(), s["tokens"], s["picks"]
    base = cu[seq]
    has = parents >= 0
    up = torch.where(has, base + parents, 0)
    wanted = has & (picks[up] == tokens)  # what its parent asks for
    # of several such children the first counts
    first = torch.full((N,), N, dtype=torch.long, device=cu.device)
    me = torch.arange(N, device=cu.device)
    first.scatter_reduce_(0, torch.where(wanted, up, 0), torch.where(wanted, me, N), "amin")
    step = first
    node = torch.where(cu[1:] > cu[:-1], cu[:-1], N)  # the root of each request, N: none
    step = torch.cat([step, step.new_full((1,), N)])
    ext = torch.cat([picks, picks.new_full((1,), -1)])
    path, nxt = [], torch.full((B,), -1, dtype=picks.dtype, device=cu.device)
    for _ in range(T):
        path.append(torch.where(node < N, node - cu[:-1], -1))
        nxt = torch.where(node < N, ext[node], nxt)
        node = step[node]
    path = torch.stack(path, 1)
    accepted = (path >= 0).sum(1)
    d = torch.arange(T, device=cu.device)[None, :]
    moves = path >= 0
    src, dst = (lens[:, None] + path)[moves], (lens[:, None] + d).expand(B, T)[moves]
    b = torch.arange(B, device=cu.device)[:, None].expand(B, T)[moves]
    page = s["k_pool"].shape[2]
    src = (s["table"].long()[b, src // page], src % page)
    dst = (s["table"].long()[b, dst // page], dst % page)
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, dst[0], dst[1]] = pool[:, src[0], src[1]]
    return {"path": path.int(), "accepted": accepted.int(), "next": nxt,
            "lens": (lens + accepted).int(), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


_PLAIN = {"plan": _plain_plan, "append": _plain_append, "tree": _plain_tree,
          "logits": _plain_logits, "commit": _plain_commit}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, request by request
# ---------------------------------------------------------------------------

def _chain(parents, i):
    """Node i and its ancestors."""
    found = []
    while i >= 0:
        found.append(i)
        i = parents[i]
    return found


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers only
    s = prepare(case, seed)
    return _EXACT[case["op"]](s)


def _exact_append(s):
    style = s["case"]["style"]
    pos, slots = s["positions"].tolist(), s["slots"].tolist()
    cos, sin = s["cos"].double()[pos], s["sin"].double()[pos]
    D = cos.shape[1] * 2
    first = list(range(0, D, 2)) if style == "norm" else list(range(D // 2))
    second = [i + 1 for i in first] if style == "norm" else [i + D // 2 for i in first]

    def turned(x):
        x = x.double()
        y = torch.empty_like(x)
        y[..., first] = x[..., first] * cos[:, None] - x[..., second] * sin[:, None]
        y[..., second] = x[..., first] * sin[:, None] + x[..., second] * cos[:, None]
        return y

    kept = [t for t, at in enumerate(slots) if at >= 0]
    at = [slots[t] for t in kept]
    k, v = s["k_pool"].double(), s["v_pool"].double()
    k.flatten(0, 1)[at] = turned(s["k"])[kept]
    v.flatten(0, 1)[at] = s["v"].double()[kept]
    return {"q": turned(s["q"]), "k_pool": k, "v_pool": v}


def _exact_tree(s):
    q = s["q"].double()
    H, D = q.shape[1:]
    KV = s["k_pool"].shape[-2]
    page = s["k_pool"].shape[1]
    cu, lens, parents = s["cu"].tolist(), s["lens"].tolist(), s["parents"].tolist()
    out = torch.empty_like(q)
    for b, ln in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if s["table"] is None:
            k, v = s["k_pool"][b, :ln + n].double(), s["v_pool"][b, :ln + n].double()
        else:
            pages = s["table"][b, :_pages(ln + n, page)].long()
            k = s["k_pool"][pages].flatten(0, 1)[:ln + n].double()
            v = s["v_pool"][pages].flatten(0, 1)[:ln + n].double()
        blind = torch.ones((n, n), dtype=torch.bool)
        for i in range(n):
            blind[i, _chain(parents[cu[b]:cu[b + 1]], i)] = False
        blind = blind.cuda()
        for g in range(KV):
            heads = slice(g * (H // KV), (g + 1) * (H // KV))
            x = q[cu[b]:cu[b + 1], heads] @ k[:, g].T / math.sqrt(D)
            x[:, :, ln:].masked_fill_(blind[:, None, :], -math.inf)
            out[cu[b]:cu[b + 1], heads] = torch.softmax(x, -1) @ v[:, g]
    return out


def _exact_logits(s):
    cu, start = s["cu"].tolist(), s["hist_start"].tolist()
    V = s["logits"].shape[1]
    parents, tokens = s["parents"].tolist(), s["tokens"].tolist()
    out = s["logits"].double()
    ids = torch.arange(V, device="cuda")
    for b in range(len(cu) - 1):
        words = s["hist"][start[b]:start[b + 1]].long()
        p = int(s["prompt_lens"][b])
        told = torch.zeros(V, dtype=torch.bool, device="cuda")
        told[words[:p]] = True
        said = torch.bincount(words[p:], minlength=V).double()
        lo, hi = s["bias_start"][b:b + 2].tolist()
        rep, pres, freq = (float(s[w][b]) for w in ("repetition", "presence", "frequency"))
        for r in range(cu[b], cu[b + 1]):
            x = out[r]
            if hi > lo:
                x[s["bias_ids"][lo:hi].long()] += s["bias"][lo:hi].double()
            c = said.clone()
            for i in _chain(parents[cu[b]:cu[b + 1]], r - cu[b]):
                c[tokens[cu[b] + i]] += 1
            again = told | (c > 0)
            x[again] = torch.where(x[again] > 0, x[again] / rep, x[again] * rep)
            x -= freq * c + pres * (c > 0)
            if s["mask"] is not None:
                word = s["mask"][r].long()[ids >> 5]
                x[((word >> (ids & 31)) & 1) == 0] = -math.inf
    return {"logits": out, "picks": None}


def _exact_commit(s):
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    tokens, picks, parents = (s[w].tolist() for w in ("tokens", "picks", "parents"))
    page, table = s["k_pool"].shape[2], s["table"].tolist()
    pools = [s["k_pool"].double(), s["v_pool"].double()]
    for b, ln in enumerate(lens):
        n, base = cu[b + 1] - cu[b], cu[b]
        at, path = 0, []
        while at is not None and n:
            path.append(at)
            at = next((i for i in range(n) if parents[base + i] == at
                       and tokens[base + i] == picks[base + at]), None)
        for pool in pools:
            rows = [pool[:, table[b][(ln + i) // page], (ln + i) % page].clone() for i in path]
            for d, x in enumerate(rows):
                pool[:, table[b][(ln + d) // page], (ln + d) % page] = x
    return {"path": None, "accepted": None, "next": None, "lens": None,
            "k_pool": pools[0], "v_pool": pools[1]}


_EXACT = {"append": _exact_append, "tree": _exact_tree, "logits": _exact_logits,
          "commit": _exact_commit}
