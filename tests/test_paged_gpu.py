"""The paged-cache and draft-tree operators (paged.py) against their
definitions in 64 bits (paged_ref.py).

Tolerances, from the operations:
- attention, 16-bit types: the output's own rounding, u |out|, and the softmax
  weights' rounding for the second product, u sum p |v| (u the type's unit
  roundoff); f32 scores differ from exact ones by less than D 2^-24 sum |q k|
  scale, about 1e-4 for unit-variance rows up to D = 256, which moves every
  weight by that share: 2e-4 sum p |v|.  f32 type: the scores' part alone.
- RoPE: the output's rounding and one f32 rounding per product and sum.
- logits: one f32 rounding per operation; the same operations in numpy's
  float32 agree bit for bit.
- bookkeeping, picks, paths, moved rows: equal.
"""
import math

import numpy as np
import pytest
import torch

from tests import paged_ref as ref
from tests.paged_ref import TDT, UNIT

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(np.asarray(x, np.int32).copy(), device=dev)


class Setup:
    """A batch of trees over random caches: device tensors and the host's view."""

    def __init__(self, dev, dt, D, H, KV, lens, nodes, page, shape="mixed", seed=0, garbage=False,
                 parents=True, q_pad=0):
        rng = np.random.default_rng(seed)
        self.rng, self.dt, self.D, self.H, self.KV = rng, dt, D, H, KV
        self.lens, self.nodes, self.page = lens, nodes, page
        B = len(lens)
        rows = [a + b for a, b in zip(lens, nodes)]
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
        self.trees = [ref.random_tree(n, rng, shape) for n in nodes]
        self.parents = sum(self.trees, []) if parents else None
        n = self.cu[-1]
        if page:
            self.table, pages = ref.deal_pages(rows, page, rng)
            dims = (pages, page, KV, D)
        else:
            self.table, dims = None, (B, max(rows + [1]) + 3, KV, D)
        fill = float("nan") if garbage else 0.0
        self.k = torch.full(dims, fill, device=dev).to(TDT[dt])
        self.v = torch.full(dims, fill, device=dev).to(TDT[dt])
        self.kh, self.vh = [], []
        for b, r in enumerate(rows):
            kb = torch.from_numpy(rng.standard_normal((r, KV, D), dtype=np.float32)).to(dev).to(TDT[dt])
            vb = torch.from_numpy(rng.standard_normal((r, KV, D), dtype=np.float32)).to(dev).to(TDT[dt])
            if page:
                at = torch.tensor([int(self.table[b, i // page]) * page + i % page for i in range(r)],
                                  device=dev, dtype=torch.long)
                self.k.view(-1, KV, D)[at] = kb
                self.v.view(-1, KV, D)[at] = vb
            else:
                self.k[b, :r], self.v[b, :r] = kb, vb
            self.kh.append(kb.double().cpu().numpy())
            self.vh.append(vb.double().cpu().numpy())
        wide = torch.from_numpy(rng.standard_normal((n, H + q_pad, D), dtype=np.float32)).to(dev).to(TDT[dt])
        self.q = wide[:, :H]
        self.dev = dict(lens=i32(lens, dev), cu=i32(self.cu, dev),
                        parents=i32(self.parents, dev) if parents else None,
                        table=i32(self.table, dev) if page else None)

    def run(self, **kw):
        from alpacca_open_sourced_by_jt_b200 import _lib, paged
        d = self.dev
        out = paged.tree_decode(kw.pop("q", self.q), self.k, self.v, d["lens"], d["cu"], d["parents"],
                                table=d["table"], max_nodes=max(self.nodes + [1]),
                                max_len=max(a + b for a, b in zip(self.lens, self.nodes)), **kw)
        _lib.raise_device_error()
        return out

    def check(self, out, lse=None, scale=None):
        scale = scale or 1.0 / math.sqrt(self.D)
        o, l, w = ref.attention(self.q.double().cpu().numpy(), self.kh, self.vh, self.lens, self.cu,
                                self.parents, scale)
        u = UNIT[self.dt] if self.dt != "f32" else 0.0
        bound = u * (np.abs(o) + w) + 2e-4 * w + 1e-7
        err = np.abs(out.double().cpu().numpy() - o)
        assert np.isfinite(err).all()
        assert (err <= bound).all(), float((err / bound).max())
        if lse is not None:
            assert np.abs(lse.double().cpu().numpy() - l).max() < 2e-4


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,KV,nodes", [(8, 8, [1, 3]), (8, 2, [2, 1]), (8, 2, [4, 3]),
                                        (16, 2, [7, 4]), (12, 4, [33, 5]), (16, 1, [20, 64])])
def test_attention_types_heads_rows(cuda_dev, dt, D, H, KV, nodes):
    s = Setup(cuda_dev, dt, D, H, KV, [150, 64], nodes, 32, seed=D + H)
    s.check(s.run())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("page", [0, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("lens,nodes", [([0], [1]), ([0, 1, 63, 64, 65], [1, 2, 1, 5, 3]),
                                        ([127, 128, 129, 700], [4, 1, 8, 2]),
                                        ([15, 16, 17, 1030], [17, 16, 15, 9])])
def test_attention_lengths_and_pages(cuda_dev, dt, page, lens, nodes):
    """Empty prefixes, single rows, tiles and pages that end inside one another."""
    s = Setup(cuda_dev, dt, 64, 8, 2, lens, nodes, page, seed=page + len(lens))
    lse = torch.empty((s.cu[-1], 8), device=cuda_dev)
    s.check(s.run(lse=lse), lse)


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("shape", ["chain", "star", "forest", "mixed"])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 128])
def test_attention_tree_shapes(cuda_dev, dt, shape, n):
    s = Setup(cuda_dev, dt, 128, 4, 2, [40], [n], 16, shape=shape, seed=n)
    s.check(s.run())
    if shape == "chain":  # no parents: the same
        full = s.run()
        s.dev["parents"] = None
        assert torch.equal(s.run(), full)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nodes", [[1, 0, 2, 1], [6, 0, 24, 5]])
def test_attention_cut_items(cuda_dev, dt, nodes):
    """Contexts long enough that items are cut between CTAs and joined; a request
    without nodes among them; head and strides of a packed projection."""
    s = Setup(cuda_dev, dt, 128, 16, 4, [5000, 300, 2111, 9], nodes, 64, seed=3, q_pad=8)
    lse = torch.empty((s.cu[-1], 16), device=cuda_dev)
    out = s.run(lse=lse)
    s.check(out, lse)
    assert torch.equal(out, s.run())  # and a rerun is bit-identical


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("bf16", 256), ("f32", 128)])
@pytest.mark.parametrize("T", [1, 2, 4, 8, 16, 40])
def test_attention_many_tiles(cuda_dev, dt, D, T):
    """Every CTA's range is many tiles long: the tile ring goes round several
    times for each count of query rows (4 to 160).  The definition in 64 bits is
    evaluated on the device."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    g = torch.Generator("cuda").manual_seed(T + D)
    B, H, KV, page = 12, 16, 4, 32
    lens = [2500 + 17 * b for b in range(B)]
    rows = [n + T for n in lens]
    rng = np.random.default_rng(T)
    table, pages = ref.deal_pages(rows, page, rng)
    k = torch.randn((pages, page, KV, D), device=cuda_dev, generator=g).to(TDT[dt])
    v = torch.randn((pages, page, KV, D), device=cuda_dev, generator=g).to(TDT[dt])
    q = torch.randn((B * T, H, D), device=cuda_dev, generator=g).to(TDT[dt])
    trees = [ref.random_tree(T, rng) for _ in range(B)]
    out = paged.tree_decode(q, k, v, i32(lens, cuda_dev), i32(np.arange(B + 1) * T, cuda_dev),
                            i32(sum(trees, []), cuda_dev), table=i32(table, cuda_dev), max_nodes=T,
                            max_len=max(rows))
    _lib.raise_device_error()
    for b in range(B):
        at = torch.from_numpy(table[b, :-(-rows[b] // page)]).long().to(cuda_dev)
        kb = k[at].flatten(0, 1)[:rows[b]].double().repeat_interleave(H // KV, 1)
        vb = v[at].flatten(0, 1)[:rows[b]].double().repeat_interleave(H // KV, 1)
        s = torch.einsum("thd,rhd->htr", q[b * T:(b + 1) * T].double(), kb) / math.sqrt(D)
        blind = torch.ones((T, T), dtype=torch.bool)
        for i in range(T):
            blind[i, ref.chain_of(trees[b], i)] = False
        s[:, :, lens[b]:].masked_fill_(blind.to(cuda_dev), -math.inf)
        p = torch.softmax(s, -1)
        o = torch.einsum("htr,rhd->thd", p, vb)
        w = torch.einsum("htr,rhd->thd", p, vb.abs())
        u = UNIT[dt] if dt != "f32" else 0.0
        err = (out[b * T:(b + 1) * T].double() - o).abs()
        assert (err <= u * (o.abs() + w) + 2e-4 * w + 1e-7).all(), b


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [0, 16, 128])
def test_attention_never_written_rows_do_not_leak(cuda_dev, dt, page):
    s = Setup(cuda_dev, dt, 64, 8, 2, [70, 129, 0, 600], [3, 9, 1, 1], page, garbage=True, seed=5)
    s.check(s.run())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_attention_scale_and_large_scores(cuda_dev, dt):
    """Scores far apart (one row takes all the weight), a scale of its own."""
    s = Setup(cuda_dev, dt, 64, 4, 2, [333], [5], 16, seed=8)
    s.check(s.run(scale=0.02), scale=0.02)
    s.k *= 32
    s.kh = [k * 32 for k in s.kh]
    out = s.run().double().cpu().numpy()
    o, _, w = ref.attention(s.q.double().cpu().numpy(), s.kh, s.vh, s.lens, s.cu, s.parents, 0.125)
    # 32 times the scores: 32 times their rounding, as a share of the weights
    u = UNIT[dt] if dt != "f32" else 0.0
    assert (np.abs(out - o) <= u * (np.abs(o) + w) + 32 * 2e-4 * w + 1e-7).all()


def test_attention_padding_rows_and_graph(cuda_dev):
    """A captured step replays for other lengths and trees; rows past cu[B] come
    out zero (lse -inf)."""
    from alpacca_open_sourced_by_jt_b200 import paged
    s = Setup(cuda_dev, "bf16", 128, 8, 2, [900, 37, 411], [6, 1, 3], 32, seed=11)
    n = 16
    q = torch.randn((n, 8, 128), device=cuda_dev).to(torch.bfloat16)
    q[:10] = s.q
    par = torch.full((n,), -1, dtype=torch.int32, device=cuda_dev)
    par[:10] = s.dev["parents"]
    out = torch.full((n, 8, 128), float("nan"), device=cuda_dev).to(torch.bfloat16)
    lse = torch.zeros((n, 8), device=cuda_dev)
    ws = paged.tree_decode_workspace(8, 8, 2, 128, torch.bfloat16, 928, cuda_dev)
    d = s.dev

    def step():
        paged.tree_decode(q, s.k, s.v, d["lens"], d["cu"], par, table=d["table"], max_nodes=8,
                          max_len=928, out=out, lse=lse, workspace=ws)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for lens, nodes in (([900, 37, 411], [6, 1, 3]), ([640, 20, 64], [2, 8, 0])):
        cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
        trees = [ref.random_tree(k, s.rng) for k in nodes]
        d["lens"].copy_(i32(lens, cuda_dev))
        d["cu"].copy_(i32(cu, cuda_dev))
        par[:cu[-1]].copy_(i32(sum(trees, []), cuda_dev))
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        t = d["table"].cpu().numpy()
        rows = [[int(t[b, i // 32]) * 32 + i % 32 for i in range(lens[b] + nodes[b])] for b in range(3)]
        kh = [s.k.reshape(-1, 2, 128)[r].double().cpu().numpy() for r in rows]
        vh = [s.v.reshape(-1, 2, 128)[r].double().cpu().numpy() for r in rows]
        o, _, w = ref.attention(q[:cu[-1]].double().cpu().numpy(), kh, vh, lens, cu, sum(trees, []),
                                128 ** -0.5)
        err = np.abs(out[:cu[-1]].double().cpu().numpy() - o)
        assert (err <= UNIT["bf16"] * (np.abs(o) + w) + 2e-4 * w).all()
        assert (out[cu[-1]:] == 0).all() and torch.isneginf(lse[cu[-1]:]).all()


def test_attention_agrees_with_decode_on_single_tokens(cuda_dev):
    """One node per request is a decode step over len + 1 rows."""
    from alpacca_open_sourced_by_jt_b200 import device
    s = Setup(cuda_dev, "bf16", 128, 32, 8, [1000, 77, 2047], [1, 1, 1], 0, seed=2)
    out = s.run()
    s.check(out)
    dec = device.decode(s.q.float().contiguous(), s.k, s.v, i32([1001, 78, 2048], cuda_dev))
    assert (out.float() - dec).abs().max().item() < 2e-2


def test_attention_long_context_offsets(cuda_dev):
    """A pool of more than 2^31 elements: rows whose offsets pass 32 bits."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    KV, D, page, H = 8, 256, 128, 16
    pages = 8256  # x 128 x 8 x 256 = 2.16e9 elements
    k = torch.zeros((pages, page, KV, D), dtype=torch.bfloat16, device=cuda_dev)
    v = torch.zeros_like(k)
    lens, n = [500], 3
    table = i32([[pages - 1, 3, pages - 2, pages - 3]], cuda_dev)
    g = torch.Generator("cuda").manual_seed(1)
    kb = torch.randn((4 * page, KV, D), device=cuda_dev, generator=g).to(torch.bfloat16)
    vb = torch.randn((4 * page, KV, D), device=cuda_dev, generator=g).to(torch.bfloat16)
    for i, p in enumerate([pages - 1, 3, pages - 2, pages - 3]):
        k[p], v[p] = kb[i * page:(i + 1) * page], vb[i * page:(i + 1) * page]
    q = torch.randn((n, H, D), device=cuda_dev, generator=g).to(torch.bfloat16)
    out = paged.tree_decode(q, k, v, i32(lens, cuda_dev), i32([0, n], cuda_dev),
                            i32([-1, 0, 0], cuda_dev), table=table, max_nodes=4)
    _lib.raise_device_error()
    o, _, w = ref.attention(q.double().cpu().numpy(), [kb[:503].double().cpu().numpy()],
                            [vb[:503].double().cpu().numpy()], lens, [0, n], [-1, 0, 0], 1 / 16)
    err = np.abs(out.double().cpu().numpy() - o)
    assert (err <= UNIT["bf16"] * (np.abs(o) + w) + 2e-4 * w).all()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_attention_records_bad_numbers(cuda_dev, dt):
    """Lengths past max_len, a page outside the pool and a parent that is not an
    earlier node are recorded; the other requests come out right."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    s = Setup(cuda_dev, dt, 64, 4, 2, [100, 50], [2, 2], 16, seed=4)
    d = s.dev
    good = s.run()

    def run(lens=None, table=None, parents=None):
        out = paged.tree_decode(s.q, s.k, s.v, lens if lens is not None else d["lens"], d["cu"],
                                parents if parents is not None else d["parents"],
                                table=table if table is not None else d["table"], max_nodes=2,
                                max_len=102)
        code, _ = _lib.device_error(clear=True)
        return out, code

    out, code = run(lens=i32([101, 50], cuda_dev))
    assert code == _lib.ERR_POSITION and torch.equal(out[2:], good[2:])
    t = d["table"].clone()
    t[0, 2] = 100000
    out, code = run(table=t)
    assert code == _lib.ERR_POSITION and torch.equal(out[2:], good[2:])
    out, code = run(parents=i32([-1, 5, -1, 0], cuda_dev))
    assert code == _lib.ERR_POSITION


# ---------------------------------------------------------------------------
# RoPE + append by slot
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("style", ["norm", "neox"])
@pytest.mark.parametrize("D,n_rot", [(64, 64), (128, 96), (256, 256), (80, 20), (66, 66), (128, 0)])
def test_rope_append_matches_definition(cuda_dev, src, dt, style, D, n_rot):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    rng = np.random.default_rng(D + n_rot)
    n, H, KV, page, pages = 13, 6, 2, 16, 4
    qkv = torch.from_numpy(rng.standard_normal((n, H + 2 * KV, D), dtype=np.float32)).to(cuda_dev).to(TDT[src])
    q, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    bias = D != 66
    bq, bk, bv = (torch.from_numpy(rng.standard_normal((m, D), dtype=np.float32)).to(cuda_dev) if bias
                  else None for m in (H, KV, KV))
    pos = rng.integers(0, 40, n)
    slots = rng.permutation(pages * page)[:n]
    slots[5] = -1
    theta = rng.standard_normal((40, max(n_rot // 2, 1)))[:, :n_rot // 2]
    cos, sin = np.cos(theta).astype(np.float32), np.sin(theta).astype(np.float32)
    if n_rot == 0:
        cos = sin = np.zeros((40, 0), np.float32)
    kp = torch.full((pages, page, KV, D), 7.0, device=cuda_dev).to(TDT[dt])
    vp = kp.clone()
    args = (q, k, v, i32(pos, cuda_dev), i32(slots, cuda_dev))
    tabs = (torch.from_numpy(cos).to(cuda_dev), torch.from_numpy(sin).to(cuda_dev))
    if n_rot == 0:  # an empty table has no address: any will do
        tabs = tuple(torch.zeros((40, 1), device=cuda_dev)[:, :0].contiguous() for _ in range(2))
        with pytest.raises(_lib.B2AError):
            paged.rope_append(*args, *tabs, k_pool=kp, v_pool=vp, style=style)
        return
    out = paged.rope_append(*args, *tabs, k_pool=kp, v_pool=vp, style=style, n_rot=n_rot, bq=bq, bk=bk, bv=bv)
    _lib.raise_device_error()
    assert out.dtype == TDT[dt]

    def host(x, b):
        x = x.double().cpu().numpy()
        return x + (b.double().cpu().numpy() if b is not None else 0.0)

    c, s = cos[pos].astype(np.float64), sin[pos].astype(np.float64)
    f32, u = 2.0 ** -24, UNIT[dt]
    for got, want, mag in ((out, ref.rotate(host(q, bq), c, s, n_rot, style), host(q, bq)),
                           (kp.view(-1, KV, D)[np.maximum(slots, 0)],
                            ref.rotate(host(k, bk), c, s, n_rot, style), host(k, bk)),
                           (vp.view(-1, KV, D)[np.maximum(slots, 0)], host(v, bv), host(v, bv))):
        e = np.abs(got.double().cpu().numpy() - want)
        if got is not out:
            e[slots < 0] = 0
        # three f32 roundings (bias, product, sum) of numbers up to twice the row's largest
        top = np.abs(mag).max(axis=-1, keepdims=True)
        assert (e <= u * np.abs(want) + 8 * f32 * top).all()
    untouched = np.setdiff1d(np.arange(pages * page), slots[slots >= 0])
    assert (kp.view(-1, KV, D)[untouched] == 7).all() and (vp.view(-1, KV, D)[untouched] == 7).all()


def test_rope_append_equals_the_contiguous_append(cuda_dev):
    """The same rows through b2a_rope_append: bit for bit."""
    from alpacca_open_sourced_by_jt_b200 import device, paged
    rng = np.random.default_rng(1)
    n, H, KV, D = 9, 8, 2, 128
    q, k, v = (torch.from_numpy(rng.standard_normal((n, m, D), dtype=np.float32)).to(cuda_dev)
               for m in (H, KV, KV))
    pos = i32(rng.permutation(64)[:n], cuda_dev)
    cos, sin = device.rope_tables(64, D, 10000.0, device=cuda_dev)
    kc = torch.zeros((1, 64, KV, D), dtype=torch.bfloat16, device=cuda_dev)
    vc = torch.zeros_like(kc)
    qo = torch.empty((n, H, D), dtype=torch.bfloat16, device=cuda_dev)
    device.rope_append(q, k, v, pos, cos, sin, k_cache=kc, v_cache=vc, q_out=qo)
    kp, vp = torch.zeros_like(kc).view(4, 16, KV, D), torch.zeros_like(kc).view(4, 16, KV, D)
    out = paged.rope_append(q, k, v, pos, pos, cos, sin, k_pool=kp, v_pool=vp)
    assert torch.equal(out, qo)
    assert torch.equal(kp.view_as(kc), kc) and torch.equal(vp.view_as(vc), vc)


def test_rope_append_records_bad_positions_and_slots(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib, device, paged
    cos, sin = device.rope_tables(16, 64, 10000.0, device=cuda_dev)
    q = torch.ones((2, 2, 64), device=cuda_dev)
    kp = torch.zeros((2, 16, 2, 64), device=cuda_dev)
    vp = torch.zeros_like(kp)
    for pos, slot in (([3, 16], [0, 1]), ([3, -1], [0, 1]), ([3, 4], [0, 32])):
        kp.zero_()
        paged.rope_append(q, q, q, i32(pos, cuda_dev), i32(slot, cuda_dev), cos, sin, k_pool=kp, v_pool=vp)
        assert _lib.device_error(clear=True)[0] == _lib.ERR_POSITION
        assert (kp[0, 0] != 0).any() and not kp.view(32, 2, 64)[1:].any()


# ---------------------------------------------------------------------------
# block tables and slot maps
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("page", [1, 16, 64])
@pytest.mark.parametrize("B,trees,short", [(1, False, 0), (7, True, 0), (40, False, 30), (300, True, 10),
                                           (600, False, 0)])
def test_page_plan_matches_definition(cuda_dev, page, B, trees, short):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    rng = np.random.default_rng(page + B)
    lens = rng.integers(0, 300, B)
    add = rng.integers(0, 129 if trees else 400, B)
    add[rng.random(B) < 0.2] = -1
    held = -(-lens // page) + (rng.random(B) < 0.3)  # pages of rejected drafts stay with a request
    wide = int(max(held.max(), (-(-(lens + np.maximum(add, 0)) // page)).max())) + 1
    if B > 5:  # one request whose rows do not fit the table
        lens[3], add[3], held[3] = wide * page, 5, wide
    need = int(np.maximum(-(-(lens + np.maximum(add, 0)) // page) - held, 0)[add >= 0].sum())
    free = max(need - short, 1)
    total = int(held.sum()) + free + 3
    perm = rng.permutation(total)
    table = np.full((B, wide), -1, np.int64)
    at = 0
    for b in range(B):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    head = int(rng.integers(0, total))
    ring = np.full(total, -7, np.int64)
    ring[(head + np.arange(free)) % total] = perm[at:at + free]
    n = int(np.maximum(add, 0).sum())
    max_tokens = n + 5
    par = None
    if trees:
        par = sum((ref.random_tree(max(int(a), 0), rng, "forest") for a in add), []) + [-1] * 5
    want = ref.plan(lens.tolist(), add.tolist(), held.tolist(), table, ring, (head, free), page,
                    max_tokens, par)
    t, r = i32(table, cuda_dev), i32(ring, cuda_dev)
    wide_table = torch.full((B, wide + 3), -1, dtype=torch.int32, device=cuda_dev)
    wide_table[:, :wide] = t
    view = wide_table[:, :wide]  # rows wider apart than max_pages
    for _ in range(2):  # a repeated call gives the same
        p = paged.page_plan(i32(lens, cuda_dev), i32(add, cuda_dev), i32(held, cuda_dev), view, r,
                            i32([head, free], cuda_dev), page_rows=page, max_tokens=max_tokens,
                            parents=i32(par, cuda_dev) if trees else None)
        _lib.raise_device_error()
        got = dict(table=view, ring=r, held=p.held, cu=p.cu, seq=p.seq, pos=p.positions, slot=p.slots,
                   state=p.ring_state)
        for key, x in got.items():
            assert np.array_equal(x.cpu().numpy(), np.asarray(want[key])), key


def test_page_plan_records_bad_numbers(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    args = dict(page_rows=16, max_tokens=8)

    def run(lens=(5, 5), add=(1, 1), held=(1, 1), parents=None):
        t = torch.zeros((2, 4), dtype=torch.int32, device=cuda_dev)
        p = paged.page_plan(i32(lens, cuda_dev), i32(add, cuda_dev), i32(held, cuda_dev), t,
                            i32(range(8), cuda_dev), i32([0, 4], cuda_dev),
                            parents=None if parents is None else i32(parents, cuda_dev), **args)
        return p, _lib.device_error(clear=True)[0]

    assert run()[1] == 0
    for kw in (dict(lens=(-1, 5)), dict(held=(9, 1)), dict(add=(1, 9)),
               dict(add=(2, 1), parents=[1, 0] + [-1] * 6)):
        assert run(**kw)[1] == _lib.ERR_POSITION, kw
    p, _ = run(lens=(-1, 5))
    assert p.slots[0].item() == -1 and p.slots[1].item() >= 0  # the other request is served


# ---------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("V", [1, 31, 1000, 4096, 4097, 32003])
@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("nodes", [[1], [9, 0, 3, 17]])
def test_constrain_logits_matches_definition(cuda_dev, V, src, dst, nodes):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    rng = np.random.default_rng(V + len(nodes))
    B = len(nodes)
    cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
    n = cu[-1]
    parents = sum((ref.random_tree(k, rng) for k in nodes), [])
    tokens = rng.integers(-1, V + 1, n)  # some outside the vocabulary
    hl = rng.integers(0, 60, B)
    hist = rng.integers(-2, min(V, 50) + 2, int(hl.sum()))
    start = np.concatenate([[0], np.cumsum(hl)]).tolist()
    prompt = [int(rng.integers(0, h + 1)) for h in hl]
    rep = rng.choice(np.array([1.0, 1.25, 0.8], np.float32), B)
    pres, freq = rng.random(B).astype(np.float32), rng.random(B).astype(np.float32)
    bias = [[(int(i), np.float32(x)) for i, x in zip(rng.integers(-1, V + 1, 6), rng.standard_normal(6) * 5)]
            for _ in range(B)]  # ids repeat: the last entry counts
    logits = torch.from_numpy((rng.standard_normal((n, V)) * 4).astype(np.float32)).to(cuda_dev).to(TDT[src])
    logits[0, V // 2] = float("-inf")
    mask = rng.random((n, V)) < 0.6
    mask[0] = True
    if n > 2:
        mask[2] = False  # nothing may follow
    words = np.zeros((n, (V + 31) // 32 + 1), np.uint32)
    for v in range(V):
        words[:, v // 32] |= mask[:, v].astype(np.uint32) << np.uint32(v % 32)
    x = logits.float().cpu().numpy()
    args = (cu, parents, tokens.tolist(), hist, start, prompt, rep, pres, freq, bias, mask)
    want = ref.constrain(x, *args)
    exact = ref.constrain(x.astype(np.float64), *args)
    out = torch.empty((n, V), dtype=TDT[dst], device=cuda_dev)
    got, picks = paged.constrain_logits(
        logits, i32(cu, cuda_dev), i32(parents, cuda_dev), i32(tokens, cuda_dev), max_nodes=20,
        hist=i32(hist, cuda_dev), hist_start=i32(start, cuda_dev), prompt_lens=i32(prompt, cuda_dev),
        repetition=torch.from_numpy(rep).to(cuda_dev), presence=torch.from_numpy(pres).to(cuda_dev),
        frequency=torch.from_numpy(freq).to(cuda_dev),
        bias_start=i32(np.arange(B + 1) * 6, cuda_dev),
        bias_ids=i32([i for r in bias for i, _ in r], cuda_dev),
        bias=torch.tensor([float(x) for r in bias for _, x in r], device=cuda_dev),
        mask=torch.from_numpy(words.view(np.int32)).to(cuda_dev), out=out)
    _lib.raise_device_error()
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(TDT[dst]))
    fine = np.isfinite(exact)
    assert np.array_equal(fine, np.isfinite(want))
    # five roundings of numbers no larger than the terms (|logit| < 30, counts < 80)
    assert np.abs(want[fine] - exact[fine]).max(initial=0.0) < 5 * 2.0 ** -24 * 128
    top = want.max(axis=1)
    lowest = np.where(np.isneginf(top), -1, (want == top[:, None]).argmax(axis=1))
    assert np.array_equal(picks.cpu().numpy(), lowest)


def test_constrain_logits_ties_zeros_nan_and_padding(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import paged
    V = 9000
    x = torch.full((6, V), -1.0, device=cuda_dev)
    x[0, 8000] = x[0, 17] = x[0, 4100] = 3.0     # equal values: the lowest token
    x[1, :] = -0.0
    x[1, 5] = 0.0                                # -0 and +0 are equal
    x[2, 3] = float("nan")                       # cannot be picked
    x[3, :] = float("-inf")
    x[3, 8999] = -3e38
    x[4, 70] = float("inf")
    cu = i32([0, 1, 2, 3, 4, 5], cuda_dev)       # row 5 is padding
    out = torch.full((6, V), 9.0, device=cuda_dev)
    _, picks = paged.constrain_logits(x, cu, None, None, max_nodes=1, out=out)
    assert picks.tolist() == [17, 0, 0, 8999, 70, -1]
    assert torch.equal(out[:5].nan_to_num(1.5), x[:5].nan_to_num(1.5)) and (out[5] == 9).all()


def test_constrain_logits_in_place_and_strided(cuda_dev):
    """Rows of odd stride (one access per logit), in place."""
    from alpacca_open_sourced_by_jt_b200 import paged
    V = 777
    wide = torch.randn((4, V + 6), device=cuda_dev)[:, 3:3 + V]
    base = wide.clone()
    cu, tok = i32([0, 2, 4], cuda_dev), i32([5, 6, 7, 8], cuda_dev)
    out, picks = paged.constrain_logits(wide, cu, None, tok, max_nodes=2, out=wide,
                                        presence=torch.full((2,), 50.0, device=cuda_dev))
    want = base.clone()
    for r, toks in enumerate(([5], [5, 6], [7], [7, 8])):
        want[r, toks] -= 50.0
    assert out is wide and torch.equal(wide, want)
    assert torch.equal(picks.long(), want.argmax(1))


def test_constrain_logits_long_history_counts(cuda_dev):
    """Counts over thousands of repeats, no penalties left out."""
    from alpacca_open_sourced_by_jt_b200 import paged
    hist = i32([7] * 5000 + [9] * 3 + [11] * 70000, cuda_dev)
    x = torch.zeros((1, 64), device=cuda_dev)
    out, _ = paged.constrain_logits(x, i32([0, 1], cuda_dev), None, None, max_nodes=1, hist=hist,
                                    hist_start=i32([0, 75003], cuda_dev), prompt_lens=i32([1000], cuda_dev),
                                    frequency=torch.ones(1, device=cuda_dev))
    assert out[0, 7] == -4000 and out[0, 9] == -3 and out[0, 11] == -70000 and out[0].sum() == -74003


# ---------------------------------------------------------------------------
# commit
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("page", [0, 16, 64])
@pytest.mark.parametrize("shape", ["mixed", "chain", "star", "forest"])
def test_tree_commit_matches_definition(cuda_dev, dt, page, shape):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    rng = np.random.default_rng(page + len(shape))
    L, KV, D = 3, 2, 64
    lens, nodes = [0, 15, 100, 31, 64], [1, 20, 128, 0, 40]
    B = len(lens)
    rows = [a + b for a, b in zip(lens, nodes)]
    cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
    parents = sum((ref.random_tree(n, rng, shape) for n in nodes), [])
    tokens = rng.integers(0, 4, cu[-1])  # siblings with equal tokens: the first counts
    picks = rng.integers(0, 4, cu[-1])
    if page:
        table, pages = ref.deal_pages(rows, page, rng)
        dims = (L, pages, page, KV, D)
    else:
        table, dims = None, (L, B, max(rows), KV, D)
    k = torch.randn(dims, device=cuda_dev).to(TDT[dt])
    v = torch.randn(dims, device=cuda_dev).to(TDT[dt])
    k0, v0 = k.clone(), v.clone()
    c = paged.tree_commit(i32(picks, cuda_dev), i32(tokens, cuda_dev), i32(parents, cuda_dev),
                          i32(cu, cuda_dev), i32(lens, cuda_dev), k, v,
                          table=i32(table, cuda_dev) if page else None, max_nodes=128,
                          max_len=max(rows))
    _lib.raise_device_error()
    want = ref.accept(picks.tolist(), tokens.tolist(), parents, cu)

    def at(b, row):
        return (int(table[b, row // page]), row % page) if page else (b, row)

    for b, (path, nxt) in enumerate(want):
        assert c.path[b].tolist() == path + [-1] * (128 - len(path))
        assert c.accepted[b].item() == len(path) and c.next_token[b].item() == nxt
        assert c.lens[b].item() == lens[b] + len(path)
        for d, i in enumerate(path):
            (p, r), (sp, sr) = at(b, lens[b] + d), at(b, lens[b] + i)
            assert torch.equal(k[:, p, r], k0[:, sp, sr]) and torch.equal(v[:, p, r], v0[:, sp, sr])
            k[:, p, r], v[:, p, r] = k0[:, p, r], v0[:, p, r]  # checked: back to what it was
    assert torch.equal(k, k0) and torch.equal(v, v0)  # nothing else moved


def test_tree_commit_records_bad_numbers(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    k = torch.randn((1, 4, 16, 2, 64), device=cuda_dev)
    v, k0 = k.clone(), k.clone()
    tok = i32([1, 1, 1], cuda_dev)
    par = i32([-1, 0, 0], cuda_dev)
    for lens, table in (([62], [[0, 1, 2, 3]]), ([15], [[0, 9, 2, 3]])):
        c = paged.tree_commit(tok, i32([1, 2, 1], cuda_dev), par, i32([0, 3], cuda_dev),
                              i32(lens, cuda_dev), k, v, table=i32(table, cuda_dev), max_nodes=3)
        assert _lib.device_error(clear=True)[0] == _lib.ERR_POSITION
        assert torch.equal(k, k0)
    assert c.accepted.item() == 2


def test_other_stream(cuda_dev):
    """Every entry runs on the stream it is given."""
    from alpacca_open_sourced_by_jt_b200 import paged
    s = Setup(cuda_dev, "bf16", 64, 8, 2, [2000, 40], [5, 2], 16, seed=1)
    want = s.run()
    d = s.dev
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q = torch.zeros_like(s.q)
        torch.cuda._sleep(2_000_000)
        q.copy_(s.q)
        out = paged.tree_decode(q, s.k, s.v, d["lens"], d["cu"], d["parents"], table=d["table"],
                                max_nodes=5, max_len=2005)
    side.synchronize()
    assert torch.equal(out, want)


def test_stream_argument_owns_what_the_call_allocates(cuda_dev):
    """A call given a busy side stream: its output and workspace come from that
    stream, so work queued on the current stream afterwards cannot be handed the
    same memory while the kernels still wait."""
    from alpacca_open_sourced_by_jt_b200 import paged
    s = Setup(cuda_dev, "bf16", 64, 8, 2, [5000, 40], [5, 2], 16, seed=1)
    want = s.run()
    d = s.dev
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        out = paged.tree_decode(s.q, s.k, s.v, d["lens"], d["cu"], d["parents"], table=d["table"],
                                max_nodes=5, max_len=5005, stream=stream)
        junk = [torch.full((1 << 16,), 7.0, device=cuda_dev) for _ in range(64)]
        side.synchronize()
        assert torch.equal(out, want)
        del junk
