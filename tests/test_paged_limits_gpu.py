"""The paged-cache and draft-tree operators at their limits: padded steps,
requests that find no pages, that end or are out of bounds, numbers that are not
finite where nothing may see them.  Definitions in paged_ref.py; bookkeeping is
equal, attention within the bounds that test_paged_gpu.py derives."""
import numpy as np
import pytest
import torch

from tests import paged_ref as ref
from tests.paged_ref import TDT, UNIT

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(np.asarray(x, np.int32).copy(), device=dev)


# ---------------------------------------------------------------------------
# page plan
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("total,max_tokens", [(1500, 3000), (2048, 2055), (1024, 5000), (4097, 9000),
                                              (1153, 2048), (0, 2500)])
def test_page_plan_trees_with_whole_tiles_of_padding(cuda_dev, total, max_tokens):
    """A captured step's arrays are longer than its tokens: a CTA's 1024 tokens may
    all be padding, with more nodes before them than a tile holds."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    rng = np.random.default_rng(total)
    page = 16
    add = []
    while sum(add) < total:
        add.append(min(int(rng.integers(1, 129)), total - sum(add)))
    add += [0, -1]
    B = len(add)
    lens = rng.integers(0, 300, B)
    held = -(-lens // page)
    wide = int((-(-(lens + np.maximum(add, 0)) // page)).max()) + 1
    free = int((-(-(lens + np.maximum(add, 0)) // page) - held).sum()) + 1
    size = int(held.sum()) + free
    perm = rng.permutation(size)
    table = np.full((B, wide), -1, np.int64)
    at = 0
    for b in range(B):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    ring = np.full(size, -7, np.int64)
    ring[(3 + np.arange(free)) % size] = perm[at:]
    par = sum((ref.random_tree(max(a, 0), rng) for a in add), []) + [-1] * (max_tokens - total)
    want = ref.plan(lens.tolist(), add, held.tolist(), table, ring, (3, free), page, max_tokens, par)
    t, r = i32(table, cuda_dev), i32(ring, cuda_dev)
    p = paged.page_plan(i32(lens, cuda_dev), i32(add, cuda_dev), i32(held, cuda_dev), t, r,
                        i32([3, free], cuda_dev), page_rows=page, max_tokens=max_tokens,
                        parents=i32(par, cuda_dev))
    _lib.raise_device_error()
    got = dict(table=t, ring=r, held=p.held, cu=p.cu, seq=p.seq, pos=p.positions, slot=p.slots,
               state=p.ring_state)
    for key, x in got.items():
        assert np.array_equal(x.cpu().numpy(), np.asarray(want[key])), key


def test_page_plan_ended_request_takes_no_pages(cuda_dev):
    """After a request ends, its lens still stands (commit returns it unchanged):
    steps that add nothing to it leave the ring alone."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    lens, held = i32([100, 20], cuda_dev), i32([7, 2], cuda_dev)
    table = i32([[0, 1, 2, 3, 4, 5, 6, -1], [7, 8, -1, -1, -1, -1, -1, -1]], cuda_dev)
    ring, state = i32(range(12), cuda_dev), i32([9, 3], cuda_dev)
    for add, want_held, want_state in (([-1, 1], [0, 2], [9, 10]), ([0, 1], [0, 2], [9, 10]),
                                       ([0, 0], [0, 2], [9, 10]), ([0, 13], [0, 3], [10, 9])):
        p = paged.page_plan(lens, i32(add, cuda_dev), held, table, ring, state, page_rows=16, max_tokens=16)
        _lib.raise_device_error()
        held, state = p.held, p.ring_state
        assert held.tolist() == want_held and state.tolist() == want_state
    assert p.slots[:13].tolist() == [table[1, r // 16].item() * 16 + r % 16 for r in range(20, 33)]


@pytest.mark.parametrize("where", ["table", "ring"])
@pytest.mark.parametrize("page", [-1, 1 << 28, 2 ** 31 - 1])
def test_page_plan_records_pages_that_are_none(cuda_dev, where, page):
    """A number in the table or the ring that no pool has: recorded, and no slot (a
    shifted one would name a row of another page)."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    t, r = [[6, 7], [3, 4]], [0, 1, 2, 5]
    if where == "table":
        t[0][1] = page
    else:
        r[0] = page
    p = paged.page_plan(i32([30, 20], cuda_dev), i32([5, 2], cuda_dev), i32([2, 2], cuda_dev),
                        i32([x + [0] for x in t], cuda_dev), i32(r, cuda_dev), i32([0, 4], cuda_dev),
                        page_rows=16, max_tokens=7)
    assert _lib.device_error(clear=True)[0] == _lib.ERR_POSITION
    first = -1 if where == "table" else 7 * 16 + 14
    last = -1 if where == "ring" else 0
    assert p.slots.tolist() == [first, first if first < 0 else first + 1] + [
        last if last < 0 else last + i for i in range(3)] + [4 * 16 + 4, 4 * 16 + 5]


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def attend(dev, dt, D, H, KV, lens, cu, parents, q, k, v, table, max_nodes, max_len, fill=float("nan")):
    """tree_decode into buffers that hold NaN: (out, lse, device error code)."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    out = torch.full((q.shape[0], H, D), fill, device=dev).to(TDT[dt])
    lse = torch.full((q.shape[0], H), fill, device=dev)
    paged.tree_decode(q, k, v, i32(lens, dev), i32(cu, dev), None if parents is None else i32(parents, dev),
                      table=None if table is None else i32(table, dev), max_nodes=max_nodes,
                      max_len=max_len, out=out, lse=lse)
    return out, lse, _lib.device_error(clear=True)[0]


@pytest.mark.parametrize("dt,D,H,KV,n", [("bf16", 64, 8, 2, 3), ("f16", 128, 16, 2, 20), ("bf16", 256, 16, 1, 9),
                                         ("f32", 128, 8, 2, 5)])
@pytest.mark.parametrize("max_len", [640, 6000])
def test_attention_rows_of_requests_left_out_are_zero(cuda_dev, dt, D, H, KV, n, max_len):
    """Too long, too many nodes, nodes past the arrays: recorded, their rows (and the
    padding behind the last node) are zeros, never what the memory held."""
    from alpacca_open_sourced_by_jt_b200 import _lib
    rng = np.random.default_rng(D + n)
    B, page = 40, 32
    nodes = [n] * B
    lens = rng.integers(0, max_len - n + 1, B).tolist()
    table, pages = ref.deal_pages([a + n for a in lens], page, rng)
    cu = (np.arange(B + 1) * n).tolist()
    g = torch.Generator("cuda").manual_seed(n)
    k = torch.randn((pages, page, KV, D), device=cuda_dev, generator=g).to(TDT[dt])
    v = torch.randn((pages, page, KV, D), device=cuda_dev, generator=g).to(TDT[dt])
    q = torch.randn((B * n + 7, H, D), device=cuda_dev, generator=g).to(TDT[dt])
    table = np.concatenate([table, np.full((B, -(-max_len // page)), -1)], 1)
    args = (q, k, v, table, n, max_len)
    good, lse0, code = attend(cuda_dev, dt, D, H, KV, lens, cu, None, *args)
    assert code == 0 and torch.isfinite(good).all()
    assert (good[B * n:] == 0).all() and torch.isneginf(lse0[B * n:]).all()

    bad_lens = list(lens)
    for b in (0, 33, 38):  # one row too long, below zero, far too long
        bad_lens[b] = {0: max_len - n + 1, 33: -1, 38: 2 ** 31 - 1}[b]
    out, lse, code = attend(cuda_dev, dt, D, H, KV, bad_lens, cu, None, *args)
    assert code == _lib.ERR_POSITION
    for b in range(B):
        rows = slice(cu[b], cu[b + 1])
        if b in (0, 33, 38):
            assert (out[rows] == 0).all() and torch.isneginf(lse[rows]).all(), b
        else:
            assert (out[rows].float() - good[rows].float()).abs().max() < 2e-2, b
    # request 5 takes request 6's nodes too (one too many), the last ends past the arrays
    odd = list(cu)
    odd[6] += 1
    odd[B] = B * n + 8
    out, lse, code = attend(cuda_dev, dt, D, H, KV, lens, odd, None, *args)
    assert code == _lib.ERR_POSITION
    for rows in (slice(odd[5], odd[6]), slice(odd[B - 1], B * n + 7)):
        assert (out[rows] == 0).all() and torch.isneginf(lse[rows]).all()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dt,D,H,KV,nodes", [("bf16", 64, 4, 2, [6, 3]), ("f16", 128, 8, 1, [2, 1]),
                                             ("bf16", 128, 8, 2, [4, 9]), ("f16", 256, 4, 2, [4, 3]),
                                             ("bf16", 256, 16, 1, [40, 7]), ("f16", 64, 16, 2, [33, 128]),
                                             ("bf16", 128, 16, 2, [128, 70]), ("f32", 64, 8, 2, [7, 128]),
                                             ("f32", 256, 4, 4, [9, 2])])
@pytest.mark.parametrize("lens,page", [([45, 0], 16), ([500, 127], 0), ([4990, 3000], 32)])
def test_attention_hidden_infinities_and_nan_stay_hidden(cuda_dev, dt, D, H, KV, nodes, lens, page):
    """A branch whose K or V rows overflowed: the nodes that do not see it are what
    they were, those that do have the infinities and NaN of the sum over their rows."""
    from tests.test_paged_gpu import Setup
    s = Setup(cuda_dev, dt, D, H, KV, lens, nodes, page, seed=D + nodes[0])
    clean = s.run()

    def put(pool, host, b, node, cols, value):
        row = lens[b] + node
        at = (int(s.table[b, row // page]), row % page) if page else (b, row)
        pool[at[0], at[1], KV - 1, cols] = value
        host[b][row, KV - 1, cols] = value

    inf, nan = float("inf"), float("nan")
    for b, n in enumerate(nodes):
        put(s.v, s.vh, b, n - 1, 3, inf)
        put(s.v, s.vh, b, n - 1, D - 1, nan)
        put(s.v, s.vh, b, n // 2, 3, -inf)
        put(s.v, s.vh, b, n // 2, slice(8, 24), inf)
        if n > 3:
            put(s.k, s.kh, b, 2, slice(0, D), nan)
            put(s.v, s.vh, b, 2, slice(0, D), nan)
    out = s.run().double().cpu().numpy()
    u = UNIT[dt] if dt != "f32" else 0.0
    with np.errstate(all="ignore"):
        o, _, w = ref.attention(s.q.double().cpu().numpy(), s.kh, s.vh, s.lens, s.cu, s.parents, D ** -0.5)
        close = np.abs(out - o) <= u * (np.abs(o) + w) + 2e-4 * w + 1e-7
    fine = np.isfinite(o)
    assert 0 < fine.sum() < fine.size and close[fine].all()
    assert np.array_equal(out[~fine], o[~fine], equal_nan=True)
    # rows that see none of it, as before to the bit
    same = np.isfinite(o).all(axis=-1)
    assert np.array_equal(out[same], clean.double().cpu().numpy()[same])


@pytest.mark.parametrize("dt,D,H,KV,lens,nodes", [
    ("bf16", 64, 32, 2, [3000, 2000, 4100], [128, 100, 128]),  # 16 blocks a head: two rounds of 8
    ("f16", 128, 32, 4, [1500, 3000, 2100, 40, 900], [128, 1, 2, 1, 1]),  # one far above the average
    ("f32", 64, 16, 2, [1100, 2500], [40, 64])])
def test_attention_cut_items_of_many_row_blocks(cuda_dev, dt, D, H, KV, lens, nodes):
    from tests.test_paged_gpu import Setup
    s = Setup(cuda_dev, dt, D, H, KV, lens, nodes, 64, seed=sum(nodes))
    lse = torch.empty((s.cu[-1], H), device=cuda_dev)
    out = s.run(lse=lse)
    s.check(out, lse)
    assert torch.equal(out, s.run())


def test_offsets_past_32_bits(cuda_dev):
    """A pool of more than 2^31 elements: append, attention of many rows and commit at
    rows whose offsets pass 32 bits."""
    from alpacca_open_sourced_by_jt_b200 import _lib, device, paged
    KV, D, page, H, pages, ln, n = 8, 256, 128, 16, 8256, 240, 70
    k = torch.zeros((pages, page, KV, D), dtype=torch.bfloat16, device=cuda_dev)
    v = torch.zeros_like(k)
    mine = [pages - 1, 2, pages - 2]
    g = torch.Generator("cuda").manual_seed(7)
    qkv = torch.randn((ln + n, H + 2 * KV, D), device=cuda_dev, generator=g)
    rows = np.arange(ln + n)
    slots = np.array(mine)[rows // page] * page + rows % page
    tree = ref.random_tree(n, np.random.default_rng(4))
    pos = list(range(ln)) + [ln + len(ref.chain_of(tree, i)) - 1 for i in range(n)]
    cos, sin = device.rope_tables(512, D, 10000.0, device=cuda_dev)
    q = paged.rope_append(qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:], i32(pos, cuda_dev), i32(slots, cuda_dev),
                          cos, sin, k_pool=k, v_pool=v)
    small_k = torch.zeros((3, page, KV, D), dtype=torch.bfloat16, device=cuda_dev)
    small_v = torch.zeros_like(small_k)
    q2 = paged.rope_append(qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:], i32(pos, cuda_dev), i32(rows, cuda_dev),
                           cos, sin, k_pool=small_k, v_pool=small_v)
    assert torch.equal(q, q2) and torch.equal(k[mine], small_k) and torch.equal(v[mine], small_v)
    assert k.view(-1, KV * D)[:, 0].count_nonzero() == (small_k.view(-1, KV * D)[:, 0] != 0).sum()
    args = (i32([ln], cuda_dev), i32([0, n], cuda_dev), i32(tree, cuda_dev))
    out = paged.tree_decode(q[ln:], k, v, *args, table=i32([mine], cuda_dev), max_nodes=n)
    kh, vh = ([x.reshape(-1, KV, D)[:ln + n].double().cpu().numpy()] for x in (small_k, small_v))
    o, _, w = ref.attention(q[ln:].double().cpu().numpy(), kh, vh, [ln], [0, n], tree, 1 / 16)
    assert (np.abs(out.double().cpu().numpy() - o) <= UNIT["bf16"] * (np.abs(o) + w) + 2e-4 * w).all()
    tokens = list(range(n))
    picks = [max([j for j in range(n) if tree[j] == i], default=-1) for i in range(n)]
    for kp, vp, t in ((k, v, mine), (small_k, small_v, [0, 1, 2])):
        c = paged.tree_commit(i32(picks, cuda_dev), i32(tokens, cuda_dev), i32(tree, cuda_dev), args[1], args[0],
                              kp, vp, table=i32([t], cuda_dev), max_nodes=n)
        assert c.accepted.item() > 5 and c.path[0, c.accepted.item() - 1].item() > c.accepted.item()
    assert torch.equal(k[mine], small_k) and torch.equal(v[mine], small_v)
    _lib.raise_device_error()


# ---------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("cu,left_out", [([0, 3, 5, 9], [2]), ([0, 6, 7, 8], [0]), ([-1, 2, 4, 8], [0]),
                                         ([0, 2, 40, 41], [1, 2]), ([0, 9, 1, 2], [0, 1])])
def test_logits_rows_of_requests_left_out_have_no_pick(cuda_dev, cu, left_out):
    """Nodes past the arrays, too many of them, starts out of order: recorded, and no
    pick comes from memory that nothing of this call wrote."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    n, V = 8, 9000
    x = torch.randn((n, V), device=cuda_dev, generator=torch.Generator("cuda").manual_seed(len(left_out)))
    for byte in (0xff, 0x7f):
        ws = torch.full((paged._logits_bytes(n, V),), byte, dtype=torch.uint8, device=cuda_dev)
        _, picks = paged.constrain_logits(x, i32(cu, cuda_dev), None, None, max_nodes=5, workspace=ws)
        assert _lib.device_error(clear=True)[0] == _lib.ERR_POSITION
        want = [-1] * n
        for b in range(3):
            if b not in left_out:
                for r in range(cu[b], cu[b + 1]):
                    want[r] = int(x[r].argmax())
        assert picks.tolist() == want


# ---------------------------------------------------------------------------
# commit
# ---------------------------------------------------------------------------

def test_commit_ends_where_nothing_could_be_picked(cuda_dev):
    """A node whose whole row is masked has pick -1: a filler token of -1 behind it is
    not accepted."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    k = torch.randn((4, 16, 2, 64), device=cuda_dev)
    v, k0 = k.clone(), k.clone()
    tokens, parents, cu = i32([5, 7, -1, 9, -1], cuda_dev), i32([-1, 0, 1, -1, 0], cuda_dev), i32([0, 3, 5], cuda_dev)
    c = paged.tree_commit(i32([7, -1, -1, -1, 3], cuda_dev), tokens, parents, cu, i32([0, 4], cuda_dev), k, v,
                          table=i32([[0, 1], [2, 3]], cuda_dev), max_nodes=3)
    assert c.accepted.tolist() == [2, 1] and c.next_token.tolist() == [-1, -1]
    assert c.path.tolist() == [[0, 1, -1], [0, -1, -1]] and c.lens.tolist() == [2, 5]
    assert torch.equal(k, k0)
    _lib.raise_device_error()


# ---------------------------------------------------------------------------
# steps of a serving loop
# ---------------------------------------------------------------------------

def serving_loop(dev, dt, others_only):
    """Four requests over ten pages of 16 rows, four steps.  Request 3 ends in the
    second step; in the third its place goes to a new one that finds one page of
    two, while requests 1 and 2 have taken pages it gave back.  With others_only the
    new request comes one step later.  Returns per step what each request has: K and V
    rows, attention rows, plan, commit."""
    from alpacca_open_sourced_by_jt_b200 import _lib, device, paged
    L, H, KV, D, page, n_pages, max_len = 2, 4, 2, 64, 16, 10, 128
    k = torch.zeros((L, n_pages, page, KV, D), device=dev).to(TDT[dt])
    v = torch.zeros_like(k)
    table = torch.zeros((4, max_len // page), dtype=torch.int32, device=dev)
    ring, state = i32([7, 2, 9, 4, 0, 1, 8, 3, 6, 5], dev), i32([0, n_pages], dev)
    lens, held = i32([0, 0, 0, 0], dev), i32([0, 0, 0, 0], dev)
    cos, sin = device.rope_tables(max_len, D, 10000.0, device=dev)
    star = [-1] + [0] * 19
    wide = [-1, 0, 0, 1, 2, 2, 4, 5]
    chains = [[i - 1 for i in range(n)] for n in (30, 45, 10, 40)]
    new = None if others_only else star
    steps = [chains, [[-1, 0, 0]] * 3 + ["end"], [wide] * 3 + [new], [[-1, 0, 0]] * 3 + [star[:10]]]
    seen = []
    for at, trees in enumerate(steps):
        if at == 2:
            lens[3] = 0
        add = [-1 if t == "end" else 0 if t is None else len(t) for t in trees]
        nodes = [max(a, 0) for a in add]
        flat = [p for t in trees if t is not None and t != "end" for p in t]
        n = len(flat)
        plan = paged.page_plan(lens, i32(add, dev), held, table, ring, state, page_rows=page,
                               max_tokens=n, parents=i32(flat, dev))
        # a request's rows are its own whatever else is in the step
        rows = [torch.randn((m, H + 2 * KV, D), device=dev,
                            generator=torch.Generator("cuda").manual_seed(100 * at + b))
                for b, m in enumerate(nodes)]
        qkv = torch.cat(rows)
        att = []
        for li in range(L):
            q = paged.rope_append(qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:], plan.positions, plan.slots,
                                  cos, sin, k_pool=k[li], v_pool=v[li])
            att.append(paged.tree_decode(q, k[li], v[li], lens, plan.cu, i32(flat, dev), table=table,
                                         max_nodes=max(nodes), max_len=max_len))
        # the path goes to a node's last child (chains: on to the end)
        tokens, picks = [], []
        for t in trees:
            if t is None or t == "end":
                continue
            tokens += list(range(len(t)))
            kids = [[j for j in range(len(t)) if t[j] == i] for i in range(len(t))]
            picks += [c[-1] if c else 999 for c in kids]
        c = paged.tree_commit(i32(picks, dev), i32(tokens, dev), i32(flat, dev), plan.cu, lens, k, v,
                              table=table, max_nodes=max(nodes), max_len=max_len)
        _lib.raise_device_error()
        lens, held, state = c.lens, plan.held, plan.ring_state
        cu = plan.cu.tolist()
        cache = []
        for b in range(4):
            r = torch.arange(lens[b].item() if held[b] > 0 else 0, device=dev)
            where = (slice(None), table[b].long()[r // page], r % page)
            cache.append((k[where].clone(), v[where].clone()))
        seen.append(dict(cache=cache, att=[[a[cu[b]:cu[b + 1]] for a in att] for b in range(4)],
                         slots=[plan.slots[cu[b]:cu[b + 1]].tolist() for b in range(4)],
                         accepted=c.accepted.tolist(), next=c.next_token.tolist(), path=c.path.tolist(),
                         lens=lens.tolist(), held=held.tolist(), state=state.tolist(), table=table.tolist()))
    return seen


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_request_without_pages_is_left_out_of_the_step(cuda_dev, dt):
    """Plan, append, attention and commit, step by step: the request that finds no
    pages changes nothing of the others' rows, and nothing of its own is counted."""
    full, others = serving_loop(cuda_dev, dt, False), serving_loop(cuda_dev, dt, True)
    assert full[0]["lens"] == [30, 45, 10, 40] and full[1]["held"] == [3, 3, 1, 0]
    step = full[2]
    assert step["held"] == [3, 4, 2, 0] and step["state"][1] == 1  # two wanted, one there
    assert step["slots"][3] == [-1] * 20 and step["accepted"][:3] == [4, 4, 4]
    for b in range(3):
        for x, y in zip(step["cache"][b], others[2]["cache"][b]):
            assert torch.equal(x, y), b
    assert step["accepted"][3] == 0 and step["next"][3] == -1 and step["lens"][3] == 0
    assert set(step["path"][3]) == {-1} and step["table"][3][:2] == [-1, -1]
    for a in step["att"][3]:
        assert a.shape[0] == 20 and (a == 0).all()
    for at in range(4):
        for key in ("accepted", "next", "lens", "held", "state"):
            assert full[at][key] == others[at][key], (at, key)
        for b in range(3):
            for x, y in zip(full[at]["cache"][b], others[at]["cache"][b]):
                assert torch.equal(x, y), (at, b)
            for x, y in zip(full[at]["att"][b], others[at]["att"][b]):
                assert (x.float() - y.float()).abs().max() < 2e-2, (at, b)
    # one step later there is a page for ten nodes
    assert full[3]["held"][3] == 1 and full[3]["accepted"][3] == 2 and full[3]["lens"][3] == 2
    for x, y in zip(full[3]["cache"][3], others[3]["cache"][3]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("paged_cache", [True, False])
def test_step_without_nodes(cuda_dev, paged_cache):
    """All requests idle: every entry takes tensors of no rows."""
    from alpacca_open_sourced_by_jt_b200 import _lib, device, paged
    B, H, KV, D, page = 3, 8, 2, 64, 32
    none = i32([], cuda_dev)
    lens, held = i32([20, 0, 32], cuda_dev), i32([1, 0, 1], cuda_dev)
    table = i32([[4, -1], [-1, -1], [0, -1]], cuda_dev)
    ring, state = i32(range(5), cuda_dev), i32([1, 3], cuda_dev)
    k = torch.randn((5, page, KV, D), device=cuda_dev)
    v = torch.randn_like(k)
    k0, v0 = k.clone(), v.clone()
    cos, sin = device.rope_tables(64, D, 10000.0, device=cuda_dev)
    plan = paged.page_plan(lens, i32([0, 0, 0], cuda_dev), held, table, ring, state, page_rows=page,
                           max_tokens=0, parents=none)
    assert plan.cu.tolist() == [0] * (B + 1) and plan.held.tolist() == [1, 0, 1]
    assert plan.ring_state.tolist() == [1, 3] and plan.slots.numel() == 0
    rows = torch.empty((0, H + 2 * KV, D), device=cuda_dev)
    q = paged.rope_append(rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:], plan.positions, plan.slots, cos,
                          sin, k_pool=k, v_pool=v)
    t = table if paged_cache else None
    att = paged.tree_decode(q, k, v, lens, plan.cu, none, table=t, max_nodes=1,
                            lse=torch.empty((0, H), device=cuda_dev))
    assert q.shape == att.shape == (0, H, D)
    out, picks = paged.constrain_logits(torch.empty((0, 500), device=cuda_dev), plan.cu, none, none, max_nodes=1)
    assert out.shape == (0, 500) and picks.shape == (0,)
    c = paged.tree_commit(picks, none, none, plan.cu, lens, k, v, table=t, max_nodes=1)
    assert c.accepted.tolist() == [0] * B and c.next_token.tolist() == [-1] * B
    assert c.lens.tolist() == [20, 0, 32] and (c.path == -1).all()
    assert torch.equal(k, k0) and torch.equal(v, v0)
    _lib.raise_device_error()


@pytest.mark.parametrize("page,n_pages,seed", [(16, 14, 0), (16, 24, 1), (64, 8, 2)])
def test_pages_over_many_steps(cuda_dev, page, n_pages, seed):
    """Requests that come, grow by trees, find no pages and end, over forty steps on a
    ring that runs short: the device's numbers are those of the definition, and no
    page is held twice or lost."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    rng = np.random.default_rng(seed)
    B, wide = 9, 12
    table, ring = np.full((B, wide), -1, np.int64), np.arange(n_pages)
    state, lens, held = [0, n_pages], [0] * B, [0] * B
    t, r, st = i32(table, cuda_dev), i32(ring, cuda_dev), i32(state, cuda_dev)
    ln, hd = i32(lens, cuda_dev), i32(held, cuda_dev)
    k = torch.zeros((n_pages, page, 1, 64), dtype=torch.bfloat16, device=cuda_dev)
    v = torch.zeros_like(k)
    unserved = 0
    for _ in range(40):
        add = [int(rng.integers(1, 40)) if rng.random() < 0.7 else 0 for _ in range(B)]
        for b in range(B):
            if held[b] and rng.random() < 0.1:
                add[b] = -1
            elif lens[b] + max(add[b], 0) > wide * page:
                add[b] = 0
        nodes = [max(a, 0) for a in add]
        trees = [ref.random_tree(m, rng) for m in nodes]
        par = sum(trees, []) + [-1] * 3
        n = sum(nodes)
        want = ref.plan(lens, add, held, table, ring, state, page, n + 3, par)
        plan = paged.page_plan(ln, i32(add, cuda_dev), hd, t, r, st, page_rows=page, max_tokens=n + 3,
                               parents=i32(par, cuda_dev))
        tokens, picks = rng.integers(0, 3, n + 3), rng.integers(0, 3, n + 3)
        paths = ref.accept(picks.tolist(), tokens.tolist(), par, want["cu"])
        c = paged.tree_commit(i32(picks, cuda_dev), i32(tokens, cuda_dev), i32(par, cuda_dev), plan.cu, ln, k, v,
                              table=t, max_nodes=128)
        _lib.raise_device_error()
        served = [m == 0 or want["slot"][want["cu"][b]] >= 0 for b, m in enumerate(nodes)]
        unserved += served.count(False)
        assert plan.slots.tolist() == want["slot"] and plan.held.tolist() == want["held"]
        assert plan.ring_state.tolist() == want["state"]
        assert c.accepted.tolist() == [len(p) if ok else 0 for (p, _), ok in zip(paths, served)]
        assert c.next_token.tolist() == [x if ok else -1 for (_, x), ok in zip(paths, served)]
        lens = [a + (len(p) if ok else 0) for a, (p, _), ok in zip(lens, paths, served)]
        assert c.lens.tolist() == lens
        table, ring, state, held = want["table"], want["ring"], want["state"], want["held"]
        ln, hd, st = c.lens, plan.held, plan.ring_state
        for b in range(B):
            if add[b] == -1:
                lens[b] = 0
                ln[b] = 0
            assert t[b, :held[b]].tolist() == table[b, :held[b]].tolist()
        free = [int(ring[(state[0] + i) % n_pages]) for i in range(state[1])]
        assert sorted(free + [int(x) for b in range(B) for x in table[b, :held[b]]]) == list(range(n_pages))
    assert unserved > 5
