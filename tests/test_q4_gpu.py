"""Normed heads and the 4-bit cache (paged.py) against their definitions (q4_ref.py).

Appended rows, codes and scales: equal, bit for bit (each f32 operation is rounded by
itself, the norm's sum is taken in 64 bits); q and 16-bit rows against 64 bits: the
rounding u |x| of the type and 8 f32 roundings of numbers up to the pair's size.

Attention, against 64 bits over the values that the pool stands for (u the unit roundoff
of the output's type, w = sum p |v|, d the largest V scale):
- u |out| for the output, 2^-11 w for the weights' rounding to f16;
- weights under f16's normal numbers are off by 2^-25 on a scale at which the largest is
  at least 1/2, times codes up to 8: 2^-21 d a row;
- scores: a product of 11 and 4 bits is exact; sums of D products of up to 16 |q| d and
  their parts taken off again lose less than 2^-19 sum |q| 16 d scale, for unit-variance
  q of D <= 256 and d < 0.6 under 256 x 0.8 x 9.6 / 16 x 2^-19 = 2.4e-4: 5e-4 w."""
import math

import numpy as np
import pytest
import torch

from tests import paged_ref as ref
from tests import q4_ref
from tests.paged_ref import TDT, UNIT

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(np.asarray(x, np.int32).copy(), device=dev)


def f32(x, dev):
    return torch.tensor(np.asarray(x, np.float32).copy(), device=dev)


# ---- append ------------------------------------------------------------------

def rows_of(dev, src, n, H, KV, D, rng, scale=1.0):
    x = torch.from_numpy((rng.standard_normal((n, H + 2 * KV, D)) * scale).astype(np.float32)).to(dev).to(TDT[src])
    return x, x[:, :H], x[:, H:H + KV], x[:, H + KV:]


def append_case(dev, D, style, n_rot, src, n, H, KV, page, seed, scale=1.0, biased=False):
    rng = np.random.default_rng(seed)
    qkv, q, k, v = rows_of(dev, src, n, H, KV, D, rng, scale)
    pages = -(-n // page) + 2
    slots = rng.permutation(pages * page)[:n].astype(np.int32)
    if n > 2:
        slots[n // 2] = -1
    pos = rng.integers(0, 500, n).astype(np.int32)
    theta = np.outer(np.arange(500), 1e4 ** (-np.arange(0, n_rot, 2) / n_rot))
    cos, sin = np.cos(theta).astype(np.float32), np.sin(theta).astype(np.float32)
    wq = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32)
    wk = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32)
    bias = [0.5 * rng.standard_normal((h, D)).astype(np.float32) for h in (H, KV, KV)] if biased else [None] * 3
    host = [t.float().cpu().numpy() + (0 if b is None else b) for t, b in zip((q, k, v), bias)]
    return dict(q=q, k=k, v=v, slots=slots, pos=pos, cos=cos, sin=sin, wq=wq, wk=wk, pages=pages, host=host,
                bias=[None if b is None else f32(b.ravel(), dev) for b in bias])


APPENDS = [  # D, style, n_rot, src, n, H, KV, page
    (64, "neox", 64, "f32", 1, 4, 2, 16),
    (128, "neox", 128, "bf16", 33, 32, 8, 64),
    (256, "neox", 256, "f16", 7, 16, 2, 32),
    (64, "norm", 64, "f16", 700, 32, 8, 16),
    (128, "norm", 48, "f32", 19, 8, 8, 16),
    (128, "neox", 64, "f32", 19, 12, 4, 128),
    (256, "norm", 16, "bf16", 5, 6, 3, 16),
    (64, "norm", 32, "bf16", 65, 5, 1, 32),
    (128, "neox", 128, "f32", 3, 40, 40, 16),
]


@pytest.mark.parametrize("dst", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,style,n_rot,src,n,H,KV,page", APPENDS)
def test_normed_rows_into_16_and_32_bits(cuda_dev, D, style, n_rot, src, n, H, KV, page, dst):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    c = append_case(cuda_dev, D, style, n_rot, src, n, H, KV, page, 11, biased=n == 19)
    dt, eps = TDT[dst], 1e-6
    kp = torch.full((c["pages"], page, KV, D), 7.0, dtype=dt, device=cuda_dev)
    vp = kp.clone()
    bq, bk, bv = c["bias"]
    q = paged.rope_append(c["q"], c["k"], c["v"], i32(c["pos"], cuda_dev), i32(c["slots"], cuda_dev),
                          f32(c["cos"], cuda_dev), f32(c["sin"], cuda_dev), k_pool=kp, v_pool=vp,
                          n_rot=n_rot, style=style, bq=bq, bk=bk, bv=bv, q_norm=f32(c["wq"], cuda_dev),
                          k_norm=f32(c["wk"], cuda_dev), eps=eps)
    _lib.raise_device_error()
    at = (c["cos"][c["pos"]], c["sin"][c["pos"]], n_rot, style)
    want_q = torch.from_numpy(q4_ref.heads32(c["host"][0], c["wq"], eps, *at)).to(dt)
    want_k = torch.from_numpy(q4_ref.heads32(c["host"][1], c["wk"], eps, *at)).to(dt)
    want_v = torch.from_numpy(c["host"][2]).to(dt)
    assert torch.equal(q.cpu(), want_q)
    kept = np.nonzero(c["slots"] >= 0)[0]
    for pool, want in ((kp, want_k), (vp, want_v)):
        expect = torch.full_like(pool.cpu(), 7.0).view(-1, KV, D)
        expect[torch.from_numpy(c["slots"][kept].astype(np.int64))] = want[torch.from_numpy(kept)]
        assert torch.equal(pool.cpu().view(-1, KV, D), expect)
    exact = q4_ref.heads64(c["host"][0], c["wq"], eps, *at)
    pair = np.abs(exact).max(-1, keepdims=True)
    assert (np.abs(q.double().cpu().numpy() - exact) <= UNIT[dst] * np.abs(exact) + 8 * 2.0 ** -24 * pair).all()


@pytest.mark.parametrize("norms", [True, False])
@pytest.mark.parametrize("D,style,n_rot,src,n,H,KV,page", APPENDS)
def test_rows_into_4_bits(cuda_dev, D, style, n_rot, src, n, H, KV, page, norms):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    c = append_case(cuda_dev, D, style, n_rot, src, n, H, KV, page, 12, biased=n == 19)
    eps = 1e-5
    pool = paged.q4_pool(c["pages"], page, KV, D, device=cuda_dev)
    pool += 0x55  # what other slots held stays
    before = pool.cpu().numpy().copy()
    wq, wk = (c["wq"], c["wk"]) if norms else (None, None)
    bq, bk, bv = c["bias"]
    slots = i32(c["slots"], cuda_dev)
    q = paged.rope_append_q4(c["q"], c["k"], c["v"], i32(c["pos"], cuda_dev), slots, f32(c["cos"], cuda_dev),
                             f32(c["sin"], cuda_dev), pool=pool, n_rot=n_rot, style=style, bq=bq, bk=bk, bv=bv,
                             q_norm=None if wq is None else f32(wq, cuda_dev),
                             k_norm=None if wk is None else f32(wk, cuda_dev), eps=eps)
    at = (c["cos"][c["pos"]], c["sin"][c["pos"]], n_rot, style)
    assert q.dtype is (torch.float16 if src == "f32" else TDT[src])
    assert torch.equal(q.cpu(), torch.from_numpy(q4_ref.heads32(c["host"][0], wq, eps, *at)).to(q.dtype))
    rows = [q4_ref.heads32(c["host"][1], wk, eps, *at), c["host"][2]]
    # the whole pool, byte for byte
    kept = np.nonzero(c["slots"] >= 0)[0]
    places = q4_ref.granule_places(D)
    want = before
    for which, x in enumerate(rows):
        code, d = q4_ref.quantize(x)
        for i in kept:
            pg, r = divmod(int(c["slots"][i]), page)
            g = want[pg, :, r // 16]
            byte, bit = places[which][r % 16, :, 0], places[which][r % 16, :, 1]
            for dim in range(D):
                g[:, byte[dim]] = (g[:, byte[dim]] & ~np.uint8(15 << bit[dim]) & 255) | (code[i, :, dim] << bit[dim]).astype(np.uint8)
            raw = d[i].view(np.uint8).reshape(KV, D // 32, 2)
            for e in (0, 1):
                g[:, places[2 + which][r % 16] + e] = raw[..., e]
    assert np.array_equal(pool.cpu().numpy(), want)
    # and read back
    for dt in TDT:
        ks, vs = paged.q4_rows(pool, slots, dtype=TDT[dt])
        for got, x in ((ks, rows[0]), (vs, rows[1])):
            y = q4_ref.values(*q4_ref.quantize(x))
            y[c["slots"] < 0] = 0
            assert torch.equal(got.cpu(), torch.from_numpy(y).to(TDT[dt]))
    _lib.raise_device_error()


def test_special_values_into_4_bits(cuda_dev):
    """Zeros, ties, saturation, infinities, NaN and numbers below f16, in V rows (stored as
    they are) and, unrotated, in K rows."""
    from alpacca_open_sourced_by_jt_b200 import paged
    D, KV, n = 64, 2, 9
    x = np.random.default_rng(0).standard_normal((n, KV, D)).astype(np.float32)
    x[0] = 0
    x[1, 0, :3], x[1, 1, 40:43] = (3, -3, 1), (-5, 5, 5)
    x[2, 0, 7], x[2, 1, 50] = 1e9, -1e9
    x[3, 0, 7], x[3, 1, 50] = np.inf, -np.inf
    x[4, 0, 31], x[4, 1, 32] = np.nan, np.nan
    x[5] *= 1e-7
    x[6] *= 3e-5
    x[7], x[8] = 65280.0, -0.0
    t = torch.from_numpy(x).to(cuda_dev)
    pool = paged.q4_pool(1, 16, KV, D, device=cuda_dev)
    slots = torch.arange(n, dtype=torch.int32, device=cuda_dev)
    tab = torch.ones((1, D // 2), device=cuda_dev)
    paged.rope_append_q4(t, t, t, torch.zeros_like(slots), slots, tab, tab * 0, pool=pool)
    code, d = q4_ref.quantize(x)
    ks, vs = (t.cpu().numpy() for t in paged.q4_rows(pool, slots))
    want = q4_ref.values(code, d).astype(np.float32)
    np.testing.assert_array_equal(vs, want)
    kept = np.arange(n) != 3  # (an infinity turned by sin 0 is NaN)
    np.testing.assert_array_equal(ks[kept], want[kept])
    assert np.isnan(ks[3, 0, :32]).all() and np.array_equal(ks[3, 0, 32:], want[3, 0, 32:])


# ---- attention -----------------------------------------------------------------

class Q4Setup:
    """A batch of trees over a random 4-bit cache; pages that nobody has, and rows behind
    the last, hold 0xff bytes (NaN scales)."""

    def __init__(self, dev, dt, D, H, KV, lens, nodes, page, shape="mixed", seed=0, size=1.0, table=True,
                 chains=False, q_pad=0):
        rng = np.random.default_rng(seed)
        self.dev, self.dt, self.D, self.H, self.KV = dev, dt, D, H, KV
        self.lens, self.nodes, self.page = lens, nodes, page
        rows = [a + b for a, b in zip(lens, nodes)]
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
        self.parents = None if chains else sum((ref.random_tree(n, rng, shape) for n in nodes), [])
        B, n = len(lens), self.cu[-1]
        if table:
            self.table, pages = ref.deal_pages(rows, page, rng)
        else:
            self.table, pages = None, B
            page = self.page = -(-max(rows + [1]) // 16) * 16 + 16
        self.kh, self.vh, self.dmax = [], [], 0.0
        granules = np.full((pages, KV, page // 16, 18 * D), 255, np.uint8)
        places = q4_ref.granule_places(D)
        for b, r in enumerate(rows):
            pad = -r % 16
            x = (rng.standard_normal((2, r + pad, KV, D)) * size).astype(np.float32)
            (kc, kd), (vc, vd) = q4_ref.quantize(x[0]), q4_ref.quantize(x[1])
            self.kh.append(q4_ref.values(kc, kd)[:r])
            self.vh.append(q4_ref.values(vc, vd)[:r])
            self.dmax = max(self.dmax, float(np.abs(vd.astype(np.float64)).max(initial=0)))
            g = q4_ref.pack(kc[None], kd[None], vc[None], vd[None])[0] if r else None
            for i in range((r + pad) // 16):
                pg = int(self.table[b, i * 16 // page]) if table else b
                one = g[:, i]
                live = min(16, r - 16 * i)
                if live < 16:  # rows behind the last
                    for which in (0, 1):
                        one[:, places[2 + which][live:].ravel()] = 255
                        one[:, places[2 + which][live:].ravel() + 1] = 255
                granules[pg, :, i * 16 % page // 16] = one
        self.pool = torch.from_numpy(granules).to(dev)
        q = rng.standard_normal((n, H * D + q_pad)).astype(np.float32)
        self.q = torch.from_numpy(q).to(dev).to(TDT[dt])[:, :H * D].unflatten(1, (H, D))
        self.max_len = max(rows + [1])
        self.args = (self.pool, i32(lens, dev), i32(self.cu, dev),
                     None if chains else i32(self.parents, dev))
        self.kw = dict(table=None if self.table is None else i32(self.table, dev), max_nodes=max(nodes + [1]))

    def run(self, **kw):
        from alpacca_open_sourced_by_jt_b200 import paged
        return paged.tree_decode_q4(self.q, *self.args, **{**self.kw, **kw})

    def check(self, out, lse=None, scale=None):
        scale = 1 / math.sqrt(self.D) if scale is None else scale
        want, l, w = ref.attention(self.q.double().cpu().numpy(), self.kh, self.vh, self.lens, self.cu,
                                   self.parents, scale)
        got = out.double().cpu().numpy()
        tol = UNIT[self.dt] * np.abs(want) + (2.0 ** -11 + 5e-4) * w + self.max_len * 2.0 ** -21 * self.dmax
        assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
        if lse is not None:
            np.testing.assert_allclose(lse.cpu().numpy(), l, atol=5e-4, rtol=2.0 ** -18)


CASES = [  # D, H, KV, lens, nodes, page, shape
    (64, 8, 2, [0], [1], 16, "mixed"),
    (128, 8, 2, [15], [1], 16, "mixed"),
    (128, 4, 4, [31, 32, 33], [1, 1, 1], 32, "mixed"),
    (64, 32, 8, [1, 500, 0, 17], [1, 1, 1, 1], 16, "mixed"),
    (256, 16, 2, [100, 3], [1, 1], 64, "mixed"),
    (256, 16, 2, [700, 3], [5, 9], 64, "mixed"),
    (128, 32, 8, [1500, 40], [1, 1], 64, "mixed"),
    (128, 12, 4, [77, 0, 640], [4, 5, 1], 16, "mixed"),          # 15 rows a head
    (64, 16, 8, [2100, 5], [8, 2], 32, "star"),                  # 16 rows, cut over CTAs
    (128, 32, 8, [130, 64, 0], [8, 3, 1], 64, "mixed"),          # 32 rows: 4 lanes a row
    (64, 32, 8, [130, 64, 0], [13, 16, 1], 16, "forest"),        # 64 rows: 2 lanes a row
    (128, 64, 8, [100, 1100], [40, 9], 128, "mixed"),            # several blocks of 128 rows
    (64, 4, 4, [300, 12, 0], [128, 1, 100], 16, "chain"),
    (128, 48, 1, [200, 10], [3, 1], 32, "mixed"),                # 48 rows to a node's head
    (64, 128, 1, [65], [2], 16, "mixed"),                        # groups of 128
    (128, 24, 8, [1, 2, 3, 4, 5, 6, 7, 8, 9], [6, 9, 1, 2, 3, 20, 1, 1, 7], 16, "mixed"),  # short items
]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D,H,KV,lens,nodes,page,shape", CASES)
def test_attention(cuda_dev, dt, D, H, KV, lens, nodes, page, shape):
    from alpacca_open_sourced_by_jt_b200 import _lib
    s = Q4Setup(cuda_dev, dt, D, H, KV, lens, nodes, page, shape, seed=len(lens) + D)
    lse = torch.empty((s.cu[-1], H), device=cuda_dev)
    s.check(s.run(lse=lse), lse)
    # a bound on the lengths that rules out whole items: the work is cut over CTAs
    s.check(s.run(max_len=max(s.max_len, 5000), table=torch.nn.functional.pad(s.kw["table"], (0, 5000 // page + 1))))
    _lib.raise_device_error()


@pytest.mark.parametrize("nodes", [1, 3, 9, 40])
def test_blocks_without_a_table_chains_and_scale(cuda_dev, nodes):
    from alpacca_open_sourced_by_jt_b200 import _lib
    s = Q4Setup(cuda_dev, "f16", 128, 8, 2, [40, 0, 333], [nodes, 1, nodes], 0, table=False, chains=True, seed=nodes,
                q_pad=64)
    s.check(s.run(scale=0.02), scale=0.02)
    _lib.raise_device_error()


@pytest.mark.parametrize("size", [1e-4, 1e-2, 50.0, 3000.0, 60000.0])
@pytest.mark.parametrize("nodes", [1, 2, 8])
def test_scales_of_any_size(cuda_dev, size, nodes):
    """V (and K) much smaller and larger than 1, the scores kept ordinary by the scale:
    weights and scales meet inside f16 whatever their sizes are."""
    s = Q4Setup(cuda_dev, "bf16", 128, 32, 8, [150, 700], [nodes, 1], 32, seed=3, size=size)
    # (bounds as above for numbers `size` times as large; scales under 2^-14 have fewer bits,
    # but they are the pool's own)
    s.check(s.run(scale=0.09 / size), scale=0.09 / size)


@pytest.mark.parametrize("nodes", [4, 8, 33])
def test_nan_reaches_only_what_sees_it(cuda_dev, nodes):
    """A NaN scale in a tree row's V block spoils this block of the rows that see the node;
    in its K block, these rows."""
    D, H, KV, page = 128, 8, 2, 16
    for which in (0, 1):
        s = Q4Setup(cuda_dev, "f16", D, H, KV, [37, 20], [nodes, 2], page, "star", seed=5)
        clean = s.run()
        row = 37 + 2  # node 2's row: seen by itself alone
        pg = int(s.table[0, row // page])
        places = q4_ref.granule_places(D)
        s.pool[pg, 1, row % page // 16, int(places[2 + which][row % 16, 2]) + 1] = 0x7f  # block 2 of KV head 1
        s.pool[pg, 1, row % page // 16, int(places[2 + which][row % 16, 2])] = 0xff
        out = s.run()
        bad = torch.isnan(out)
        expect = torch.zeros_like(bad)
        expect[2, 4:, 64:96 if which else D] = True
        if not which:
            expect[2, 4:] = True
        assert torch.equal(bad, expect)
        assert torch.equal(out[~bad], clean[~bad])


def test_requests_left_out_padding_and_errors(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    for nodes in (1, 8, 30):
        s = Q4Setup(cuda_dev, "bf16", 64, 8, 2, [100, 50, 70], [nodes] * 3, 16, seed=9)
        want = s.run()
        cu = s.cu[-1]
        # padding rows behind the last node
        q = torch.cat([s.q, torch.ones((5, 8, 64), dtype=s.q.dtype, device=cuda_dev)])
        par = torch.cat([s.args[3], torch.zeros(5, dtype=torch.int32, device=cuda_dev)])
        out = torch.full((cu + 5, 8, 64), 9.0, dtype=torch.bfloat16, device=cuda_dev)
        lse = torch.empty((cu + 5, 8), device=cuda_dev)
        paged.tree_decode_q4(q, s.args[0], s.args[1], s.args[2], par, **s.kw, out=out, lse=lse)
        assert torch.equal(out[:cu], want) and (out[cu:] == 0).all() and (lse[cu:] == -math.inf).all()
        # a request without its last page is left out
        t = s.kw["table"].clone()
        t[1, (50 + nodes - 1) // 16:] = -1
        got = s.run(table=t)
        _lib.raise_device_error()
        assert (got[nodes:2 * nodes] == 0).all()
        assert torch.equal(got[:nodes], want[:nodes]) and torch.equal(got[2 * nodes:], want[2 * nodes:])
        # a page outside the pool inside a request is recorded
        t = s.kw["table"].clone()
        t[1, 0] = 10 ** 6
        got = s.run(table=t)
        assert _lib.device_error(clear=True) == (_lib.ERR_POSITION, 1)
        assert torch.equal(got[:nodes], want[:nodes]) and torch.equal(got[2 * nodes:], want[2 * nodes:])
        # a length out of bounds: the request is left out, and recorded
        lens = s.args[1].clone()
        lens[2] = 10 ** 6
        got = paged.tree_decode_q4(s.q, s.args[0], lens, *s.args[2:], **s.kw)
        assert _lib.device_error(clear=True)[0] == _lib.ERR_POSITION
        assert (got[2 * nodes:] == 0).all() and torch.equal(got[:2 * nodes], want[:2 * nodes])
        # the table names one page twice (a shared prefix): both are read
        t = s.kw["table"].clone()
        t[1, 1] = t[1, 0]
        got = s.run(table=t)
        s.kh[1] = np.concatenate([s.kh[1][:16], s.kh[1][:16], s.kh[1][32:]])
        s.vh[1] = np.concatenate([s.vh[1][:16], s.vh[1][:16], s.vh[1][32:]])
        s.check(got)


@pytest.mark.parametrize("nodes", [1, 8])
def test_long_contexts_cut_over_all_ctas(cuda_dev, nodes):
    """Against torch in 64 bits, request by request: 20 to 40 thousand rows, ragged."""
    D, H, KV, page = 64, 8, 2, 16
    s = Q4Setup(cuda_dev, "f16", D, H, KV, [20011, 3], [nodes, 1], page, seed=21)
    s.check(s.run())


def test_streams_graphs_and_two_calls_at_once(cuda_dev):
    """Two captured calls with workspaces of their own on two streams, replayed together,
    give what eager calls give; new lengths are read at the replay."""
    from alpacca_open_sourced_by_jt_b200 import paged
    a = Q4Setup(cuda_dev, "bf16", 128, 32, 8, [3000, 1500], [1, 1], 64, seed=1)
    b = Q4Setup(cuda_dev, "bf16", 128, 32, 8, [2500, 400], [6, 3], 64, seed=2)
    want = [a.run(), b.run()]
    streams = [torch.cuda.Stream(cuda_dev) for _ in range(2)]
    graphs, outs = [], []
    for s, st in zip((a, b), streams):
        ws = paged.tree_decode_q4_workspace(s.kw["max_nodes"], s.H, s.KV, s.D, s.kw["table"].shape[1] * 64, cuda_dev)
        out = torch.empty_like(s.q)
        s.run(out=out, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.run(out=out, workspace=ws)
        graphs.append(g)
        outs.append((out, ws))
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (out, _), w in zip(outs, want):
        assert torch.equal(out, w)
    a.args[1][0] = 1000
    a.lens[0] = 1000
    a.kh[0], a.vh[0] = a.kh[0][:1001], a.vh[0][:1001]
    graphs[0].replay()
    torch.cuda.synchronize()
    a.check(outs[0][0])
    eager = b.run(stream=streams[1])
    streams[1].synchronize()
    assert torch.equal(eager, want[1])


# ---- commit -------------------------------------------------------------------------

@pytest.mark.parametrize("D,KV,page,layers,table", [(64, 2, 16, 1, True), (128, 8, 64, 3, True), (256, 1, 32, 2, True),
                                                    (128, 3, 48, 2, False)])
def test_commit_moves_rows(cuda_dev, D, KV, page, layers, table):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    rng = np.random.default_rng(D)
    lens, nodes = [30, 0, 100, 7], [20, 1, 33, 128]
    rows = [a + b for a, b in zip(lens, nodes)]
    B = len(lens)
    cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
    parents = sum((ref.random_tree(n, rng) for n in nodes), [])
    tokens = rng.integers(0, 5, cu[-1])
    picks = rng.integers(0, 5, cu[-1])
    if table:
        tab, pages = ref.deal_pages(rows, page, rng)
    else:
        tab, pages, page = None, B, -(-max(rows) // 16) * 16
    pool = torch.from_numpy(rng.integers(0, 256, (layers, pages, KV, page // 16, 18 * D), dtype=np.uint8)).to(cuda_dev)
    pool &= 0xbf  # (no NaN scales: rows are compared as values)
    before = [q4_ref.unpack(x) for x in pool.cpu().numpy()]
    c = paged.tree_commit_q4(i32(picks, cuda_dev), i32(tokens, cuda_dev), i32(parents, cuda_dev), i32(cu, cuda_dev),
                             i32(lens, cuda_dev), pool, table=None if tab is None else i32(tab, cuda_dev),
                             max_nodes=128)
    _lib.raise_device_error()
    found = ref.accept(picks, tokens, parents, cu)

    def at(b, r):
        return (int(tab[b, r // page]), r % page) if tab is not None else (b, r)

    want = [[x.copy() for x in kv] for kv in before]
    for b, (path, nxt) in enumerate(found):
        assert c.path[b].tolist() == path + [-1] * (128 - len(path))
        assert c.accepted[b].item() == len(path) and c.next_token[b].item() == nxt
        assert c.lens[b].item() == lens[b] + len(path)
        for layer in range(layers):
            for which in range(4):
                for d, node in enumerate(path):
                    want[layer][which][at(b, lens[b] + d)] = before[layer][which][at(b, lens[b] + node)]
    for layer in range(layers):
        for got, x in zip(q4_ref.unpack(pool[layer].cpu().numpy()), want[layer]):
            assert np.array_equal(got, x)


# ---- refusals by the wrappers ------------------------------------------------------------

def test_wrappers_refuse(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    s = Q4Setup(cuda_dev, "f16", 64, 8, 2, [20], [2], 32)
    Bad = _lib.B2AShapeError
    for kw in (dict(table=s.kw["table"].long()), dict(max_nodes=0), dict(max_nodes=129), dict(scale=0.0),
               dict(scale=math.nan), dict(max_len=10 ** 6), dict(out=torch.empty((2, 8, 64), device=cuda_dev)),
               dict(max_len=2000, table=torch.zeros((1, 200), dtype=torch.int32, device=cuda_dev),
                    workspace=torch.empty(16, dtype=torch.uint8, device=cuda_dev)),
               dict(workspace=torch.empty(1 << 20, dtype=torch.uint8))):
        with pytest.raises(Bad):
            s.run(**kw)
    q, rest = s.q, s.args
    for bad_q in (q.float(), q[:, :7], q.transpose(1, 2), q.cpu()):
        with pytest.raises(Bad):
            paged.tree_decode_q4(bad_q, *rest, **s.kw)
    for bad_pool in (s.pool.float(), s.pool[..., :100], s.pool[0], s.pool.permute(0, 2, 1, 3)):
        with pytest.raises(Bad):
            paged.tree_decode_q4(q, bad_pool, *rest[1:], **s.kw)
    with pytest.raises(Bad):
        paged.q4_pool(4, 24, 2, 64, device=cuda_dev)
    with pytest.raises(Bad):
        paged.q4_pool(4, 16, 2, 80, device=cuda_dev)
    n = 3
    x, q, k, v = rows_of(cuda_dev, "f32", n, 8, 2, 64, np.random.default_rng(0))
    tab = torch.ones((4, 32), device=cuda_dev)
    pos = torch.zeros(n, dtype=torch.int32, device=cuda_dev)
    w = torch.ones(64, device=cuda_dev)
    ok = dict(pool=s.pool, q_norm=w, k_norm=w)
    paged.rope_append_q4(q, k, v, pos, pos - 1, tab, tab, **ok)
    for args, kw in (((q, k, v, pos, pos, tab[:, :8].contiguous(), tab[:, :8].contiguous()), dict(n_rot=16, style="neox")),  # not of whole blocks
                     ((q, k, v, pos, pos, tab[:, :4].contiguous(), tab[:, :4].contiguous()), {}), ((q, k, v, pos, pos.long(), tab, tab), {}),
                     ((q.half(), k, v, pos, pos, tab, tab), {}), ((q, k, v, pos, pos, tab, tab), dict(q_norm=w[:32])),
                     ((q, k, v, pos, pos, tab, tab), dict(q_out=torch.empty((n, 8, 64), device=cuda_dev))),
                     ((q, k, v, pos, pos, tab, tab), dict(eps=-1.0))):
        with pytest.raises(Bad):
            paged.rope_append_q4(*args, **{**ok, **kw})
    kp = torch.zeros((2, 16, 2, 64), device=cuda_dev)
    with pytest.raises(Bad):  # with norms q_out is of the pools' type
        paged.rope_append(q, k, v, pos, pos, tab, tab, k_pool=kp, v_pool=kp, q_norm=w,
                          q_out=torch.empty((n, 8, 64), dtype=torch.float16, device=cuda_dev))
    # a slot past the pool, a position past the table: recorded, nothing written
    before = s.pool.clone()
    paged.rope_append_q4(q, k, v, pos, pos + 10 ** 6, tab, tab, **ok)
    assert _lib.device_error(clear=True)[0] == _lib.ERR_POSITION
    paged.rope_append_q4(q, k, v, pos + 4, pos, tab, tab, **ok)
    assert _lib.device_error(clear=True)[0] == _lib.ERR_POSITION
    ks, _ = paged.q4_rows(s.pool, pos + 10 ** 6)
    assert _lib.device_error(clear=True)[0] == _lib.ERR_POSITION and (ks == 0).all()
    assert torch.equal(before, s.pool)
    # nothing to do
    assert paged.tree_decode_q4(s.q[:0], s.pool, s.args[1], torch.zeros_like(s.args[2]), None, **s.kw).shape[0] == 0
    assert paged.rope_append_q4(q[:0], k[:0], v[:0], pos[:0], pos[:0], tab, tab, **ok).shape[0] == 0
    assert paged.q4_rows(s.pool, pos[:0])[0].shape == (0, 2, 64)
