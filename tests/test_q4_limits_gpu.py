"""Attention over the 4-bit cache (paged.tree_decode_q4) at its limits, against 64 bits
over the values that the pool stands for: rows of pages outside the pool, V blocks of
unlike sizes beside one another, long contexts in which every granule of 16 rows counts.

Bounds (u the unit roundoff of the output's type, w = sum p |v|): u |out| for the output,
half a step of the type's least numbers where that is more;
2^-11 w for the weights' rounding; 5e-4 w for the scores (test_q4_gpu.py derives it for
q and K of unit variance); and where a weight's product with its block's scale is under
f16's normal numbers, 2^-25 of a scale at which the largest such product of the block is
at least 1/2, times codes up to 8:  2^-21 max(p d) a row, d the block's own scale."""
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


LEAST = {"f16": 2.0 ** -25, "bf16": 0.0}  # half a step of f16's least numbers


class Batch:
    """Trees over a 4-bit cache of given rows: k, v per request (len + nodes, KV, D)."""

    def __init__(self, dev, dt, H, k, v, nodes, page, seed=0, shape="mixed", scale=None):
        rng = np.random.default_rng(seed)
        self.dt, self.H = dt, H
        _, self.KV, self.D = k[0].shape
        rows = [len(x) for x in k]
        self.nodes, self.lens, self.page = nodes, [r - n for r, n in zip(rows, nodes)], page
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
        self.parents = sum((ref.random_tree(n, rng, shape) for n in nodes), [])
        self.table, pages = ref.deal_pages(rows, page, rng)
        self.kh, self.vh, self.vd = [], [], []
        pool = np.full((pages, self.KV, page // 16, 18 * self.D), 255, np.uint8)  # NaN scales
        for b, r in enumerate(rows):
            pad = [(0, -r % 16), (0, 0), (0, 0)]
            (kc, kd), (vc, vd) = (q4_ref.quantize(np.pad(np.asarray(x[b], np.float32), pad)) for x in (k, v))
            self.kh.append(q4_ref.values(kc, kd)[:r])
            self.vh.append(q4_ref.values(vc, vd)[:r])
            self.vd.append(np.abs(vd.astype(np.float64))[:r])
            g = q4_ref.pack(kc[None], kd[None], vc[None], vd[None])[0]
            for i in range(g.shape[1]):
                pool[self.table[b, i * 16 // page], :, i * 16 % page // 16] = g[:, i]
        self.pool = torch.from_numpy(pool).to(dev)
        self.q = torch.from_numpy(rng.standard_normal((self.cu[-1], H, self.D)).astype(np.float32)).to(dev).to(TDT[dt])
        self.scale = 1 / math.sqrt(self.D) if scale is None else scale
        self.args = (self.pool, i32(self.lens, dev), i32(self.cu, dev), i32(self.parents, dev))
        self.kw = dict(table=i32(self.table, dev), max_nodes=max(nodes), scale=self.scale)

    def run(self, q=None, **kw):
        from alpacca_open_sourced_by_jt_b200 import paged
        return paged.tree_decode_q4(self.q if q is None else q, *self.args, **{**self.kw, **kw})

    def outputs(self, **kw):
        lse = torch.empty(self.q.shape[:2], device=self.q.device)
        out = self.run(lse=lse, **kw)
        return out.double().cpu().numpy(), lse.double().cpu().numpy()

    def check(self, out, lse):
        q, group = self.q.double().cpu().numpy(), self.H // self.KV
        for b, ln in enumerate(self.lens):
            c0, n, rows = self.cu[b], self.nodes[b], self.lens[b] + self.nodes[b]
            sees = np.ones((n, rows), bool)
            for i in range(n):
                sees[i, ln:] = np.isin(np.arange(n), ref.chain_of(self.parents[c0:c0 + n], i))
            for g in range(self.KV):
                heads = slice(g * group, (g + 1) * group)
                k, v, d = (np.ascontiguousarray(x[b][:, g]) for x in (self.kh, self.vh, self.vd))
                s = np.where(sees[:, None], q[c0:c0 + n, heads] @ k.T * self.scale, -np.inf)
                top = s.max(-1, keepdims=True)
                p = np.exp(s - top)
                z = p.sum(-1, keepdims=True)
                p /= z
                want, w = p @ v, p @ np.abs(v)
                most = np.stack([(p * d[:, j]).max(-1) for j in range(d.shape[1])], -1)
                tol = UNIT[self.dt] * np.abs(want) + (2.0 ** -11 + 5e-4) * w + rows * 2.0 ** -21 * most.repeat(32, -1) + LEAST[self.dt]
                off = np.abs(out[c0:c0 + n, heads] - want)
                assert (off <= tol).all(), (b, g, float((off / np.maximum(tol, 1e-300)).max()))
                at = lse[c0:c0 + n, heads] - (top + np.log(z))[..., 0]
                assert (np.abs(at) <= 5e-4 + 2.0 ** -18 * np.abs(top[..., 0])).all(), np.abs(at).max()


def normal(rng, rows, KV, D):
    return [rng.standard_normal((r, KV, D)).astype(np.float32) for r in rows]


# ---- pages outside the pool ------------------------------------------------------

@pytest.mark.parametrize("H,KV,D", [(8, 2, 64), (16, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("nodes", [1, 3, 8, 30])
def test_rows_of_pages_outside_the_pool_are_zeros(cuda_dev, H, KV, D, nodes):
    """However many nodes there are: score 0, nothing added, and an error recorded."""
    from alpacca_open_sourced_by_jt_b200 import _lib
    rng = np.random.default_rng(nodes)
    page = 16
    rows = [60 + nodes, 95 + nodes, 21 + nodes]
    s = Batch(cuda_dev, "f16", H, normal(rng, rows, KV, D), normal(rng, rows, KV, D), [nodes] * 3, page, seed=2)
    clean = s.outputs()
    _lib.raise_device_error()
    last = (rows[1] - 1) // page
    for bad in ([0], [1, 2, 4], [last], list(range(last + 1))):
        table = s.table.copy()
        table[1, bad] = [(10 ** 6, -7, len(s.pool))[i % 3] for i in range(len(bad))]
        out, lse = s.outputs(table=i32(table, cuda_dev))
        assert _lib.device_error(clear=True) == (_lib.ERR_POSITION, 1)
        kept = s.kh[1].copy(), s.vh[1].copy(), s.vd[1].copy()
        for x in (s.kh, s.vh, s.vd):
            x[1] = x[1].copy()
            x[1][np.isin(np.arange(rows[1]) // page, bad)] = 0
        s.check(out, lse)
        s.kh[1], s.vh[1], s.vd[1] = kept
        for a, b in ((out, clean[0]), (lse, clean[1])):  # the others are as they were
            assert np.array_equal(a[:nodes], b[:nodes]) and np.array_equal(a[2 * nodes:], b[2 * nodes:])
        if len(bad) == last + 1:
            assert (out[nodes:2 * nodes] == 0).all() and np.isfinite(lse).all()


# ---- scales ------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D,H,nodes", [(64, 8, 1), (128, 8, 1), (128, 8, 4), (256, 4, 1), (256, 4, 3), (128, 8, 16)])
def test_blocks_of_unlike_sizes(cuda_dev, dt, D, H, nodes):
    """A block's outputs are as near whatever the blocks beside it hold: all rows' first
    block large, one key's alone, every key's blocks of a size of their own, blocks of
    zeros."""
    rng = np.random.default_rng(D + nodes)
    KV, rows = 2, [1500, 333 + nodes]
    k = normal(rng, rows, KV, D)
    for kind in ("first", "outlier", "all", "zeros"):
        v = normal(rng, rows, KV, D)
        for x in v:
            blocks = x.reshape(len(x), KV, D // 32, 32)
            if kind == "first":
                blocks[:, :, 0] *= 1e4
                blocks[:, :, 1] *= 1e-2
            elif kind == "outlier":
                blocks[:, :, 1] *= 1e-2
                blocks[len(x) // 3, :, 0] = 6e4
            elif kind == "all":
                blocks *= 10.0 ** rng.uniform(-3, 4, (1, 1, D // 32, 1))
            else:
                blocks[:, :, 0] *= 1e4
                blocks[:, :, 1] = 0
                blocks[7, :, 1] = 1e-2
        # (the largest values end at 65280: f16 outputs stay finite)
        for x in v:
            np.clip(x, -6e4, 6e4, out=x)
        s = Batch(cuda_dev, dt, H, k, v, [nodes, nodes], 32, seed=3)
        s.check(*s.outputs())


@pytest.mark.parametrize("D,H,nodes", [(64, 8, 1), (128, 8, 4), (256, 8, 1), (256, 4, 3), (128, 8, 16)])
def test_dims_without_values(cuda_dev, D, H, nodes):
    """Every other dim's codes stand for 0 in blocks with large scales.  With few query rows
    codes are f16 subnormals c 2^-24 or c 2^-20: an MMA lines its products up by the encoded
    exponent 2^-14 and keeps 23 bits of that, 2^-13 or 2^-17 of sum w in codes; 8 sum w, of
    normal numbers, is taken off: 2^-13 of sum p d in all, a tenth more for the accumulators'
    own 24 bits.  With more rows the cache's values are multiplied: 0."""
    for rows in (9 + nodes, 41, 300, 3000):
        rng = np.random.default_rng(rows)
        k, v = normal(rng, [rows], 2, D), normal(rng, [rows], 2, D)
        v[0][..., 1::2] = 0
        v[0][..., ::32] = 8 * rng.uniform(1, 2, (rows, 2, D // 32))
        s = Batch(cuda_dev, "bf16", H, k, v, [nodes], 16, seed=rows)
        assert (s.vh[0][..., 1::2] == 0).all()
        out, lse = s.outputs()
        q, group = s.q.double().cpu().numpy(), H // 2
        for i in range(nodes):
            at = list(range(s.lens[0])) + [s.lens[0] + j for j in ref.chain_of(s.parents, i)]
            for h in range(H):
                p = np.exp(s.kh[0][at, h // group] @ q[i, h] * s.scale)
                much = ((p / p.sum()) @ s.vd[0][at, h // group]).repeat(32)[1::2]
                room = 0 if nodes * group > 16 and D < 256 else 1.1 * 2.0 ** -13
                assert (np.abs(out[i, h, 1::2]) <= room * much).all()


# ---- long contexts -------------------------------------------------------------------

LONG = [  # D, H, KV, rows, nodes, page: query rows a KV head
    (64, 8, 2, [20012, 3, 31007], [1, 1, 1], 16),       # 4
    (128, 8, 2, [24577, 4096], [1, 1], 64),
    (64, 8, 2, [20015, 9000], [4, 2], 32),              # 16
    (128, 16, 2, [16385, 40], [8, 3], 16),              # 64: two lanes a row
    (64, 8, 2, [20019, 3], [8, 1], 16),                 # 32: four
    (128, 16, 2, [15000, 700], [16, 2], 128),           # 128: one
    (256, 8, 2, [20001], [1], 64),
    (256, 8, 2, [9001, 30], [5, 2], 16),                # 20, by blocks of 8
]


@pytest.mark.parametrize("D,H,KV,rows,nodes,page", LONG)
def test_every_granule_of_a_long_context_counts(cuda_dev, D, H, KV, rows, nodes, page):
    """V is zero but for one dim of each row, the granule's number modulo D: a granule that
    were left out, or taken twice, would change a sum over some 20 to 150 of them, all of
    one sign, by more than the bound's 1e-3 of it."""
    from alpacca_open_sourced_by_jt_b200 import _lib
    rng = np.random.default_rng(D + rows[0])
    k = normal(rng, rows, KV, D)
    v = []
    for r in rows:
        x = np.zeros((r, KV, D), np.float32)
        x[np.arange(r), :, np.arange(r) // 16 % D] = -rng.uniform(0.5, 1.5, (r, KV))
        v.append(x)
    s = Batch(cuda_dev, "bf16" if D == 128 else "f16", H, k, v, nodes, page, seed=1)
    out, lse = s.outputs()
    s.check(out, lse)
    assert (out[0] < -1e-5).all() and len({float(x) for x in s.vd[0].ravel()}) > 10
    # the bound tells a lost granule: without any one of them some sum is off by more
    q = s.q.double().cpu().numpy()
    p = np.exp(s.kh[0][:, 0] @ q[0, 0] * s.scale)
    p[s.lens[0] + 1:] = 0
    p /= p.sum()
    own = np.zeros(D)
    part = np.add.reduceat(-p * s.vh[0][:, 0].sum(-1), np.arange(0, rows[0], 16))
    np.add.at(own, np.arange(len(part)) % D, part)
    whole = -(-(s.lens[0] + 1) // 16) - 1  # (granules of the prefix)
    share = part[:whole] / own[np.arange(whole) % D]
    small = rows[0] * 2.0 ** -21 * (p[:, None] * s.vd[0][:, 0]).max() / own.min()
    assert share.min() > 2 * (UNIT[s.dt] + 2.0 ** -11 + 5e-4 + small), (share.min(), small)
    for _ in range(5):  # and is the same, call after call
        again = s.outputs()
        assert np.array_equal(again[0], out) and np.array_equal(again[1], lse)
    _lib.raise_device_error()
