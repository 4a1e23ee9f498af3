"""Sampled verification (paged.verify_picks) against its definition in 64 bits, node by
node (q4_ref.verify): equal picks.

The kernel's decisions compare sums of 32-bit exponentials (2^-21) of which at most 15
sixteenths have been taken off, and its draw 64-bit sums; inputs whose decisions lie
within 2e-5, or whose draw lies within 1e-11, of their borders are drawn anew by their
seed before the kernel runs."""
import numpy as np
import pytest
import torch

from tests import paged_ref as ref
from tests import q4_ref
from tests.paged_ref import TDT

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(np.asarray(x, np.int32).copy(), device=dev)


def f32(x, dev):
    return torch.tensor(np.asarray(x, np.float32).copy(), device=dev)


def make(nodes, V, dt, draft, shape, rng, heat=(0.7, 1.0, 0.0, 1.4), agree=0.7):
    """Logits, trees and numbers on the host; rows of dt's values."""
    n = sum(nodes)
    cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
    parents = sum((ref.random_tree(k, rng, shape) for k in nodes), [])
    x = torch.from_numpy((2.5 * rng.standard_normal((n, V))).astype(np.float32)).to(TDT[dt]).float().numpy()
    # likely tokens, some of them twice among siblings, some out of range
    tokens = np.zeros(n, np.int64)
    for b, k in enumerate(nodes):
        for i in range(k):
            p = parents[cu[b] + i]
            row = x[cu[b] + max(p, 0)]
            tokens[cu[b] + i] = (int(rng.choice(np.argsort(-row)[:4])) if rng.random() < agree
                                 else int(rng.integers(-1, V + 1)))
    q = None
    if draft:
        y = x + 0.7 * rng.standard_normal((n, V)).astype(np.float32)
        e = np.exp(y - y.max(1, keepdims=True))
        q = (e / e.sum(1, keepdims=True)).astype(np.float32)
    T = None if heat is None else np.array([heat[b % len(heat)] for b in range(len(nodes))], np.float32)
    return dict(x=x, cu=cu, parents=parents, tokens=tokens, u=rng.random(n).astype(np.float32),
                d=rng.random(len(nodes)).astype(np.float32), T=T, q=q)


def run(dev, c, dt, pad=0, max_nodes=128, shift=0, **kw):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    n, V = c["x"].shape
    wide = torch.zeros((n + pad, V + shift), device=dev).to(TDT[dt])
    wide[:n, shift:] = torch.from_numpy(c["x"]).to(dev).to(TDT[dt])
    q = None
    if c["q"] is not None:
        q = torch.zeros((n + pad, V), device=dev)
        q[:n] = f32(c["q"], dev)
    zeros = np.zeros(pad)
    out = paged.verify_picks(wide[:, shift:], i32(c["cu"], dev),
                             None if c["parents"] is None else i32(np.concatenate([c["parents"], zeros]), dev),
                             i32(np.concatenate([c["tokens"], zeros]), dev), f32(np.concatenate([c["u"], zeros]), dev),
                             f32(c["d"], dev), max_nodes=max_nodes, draft=q,
                             temperature=None if c["T"] is None else f32(c["T"], dev), **kw)
    _lib.raise_device_error()
    return out.cpu().numpy()


def wanted(c):
    return q4_ref.verify(c["x"], c["cu"], c["parents"], c["tokens"], c["u"], c["d"], c["T"], c["q"])


def settled(make_one):
    """The first case whose decisions are clear, and its picks."""
    for seed in range(50):
        c = make_one(np.random.default_rng(seed))
        picks, margin, drawn = wanted(c)
        if margin > 2e-5 and drawn > 1e-11:
            return c, picks
    raise AssertionError("no clear case")


NODES = [[1], [5, 1, 9], [1, 1, 0, 1], [128], [40, 0, 3], [2] * 40]


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nodes", NODES, ids=[str(x)[:12] for x in NODES])
@pytest.mark.parametrize("V,shift", [(1, 0), (33, 0), (1024, 0), (5003, 0), (5003, 1), (40000, 0)])
def test_picks(cuda_dev, draft, dt, nodes, V, shift):
    if V > 6000 and sum(nodes) > 60:
        V = 20001
    c, want = settled(lambda rng: make(nodes, V, dt, draft, "mixed", rng))
    assert np.array_equal(run(cuda_dev, c, dt, pad=3, shift=shift)[:sum(nodes)], want)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("nodes", [[2], [1, 2, 0, 2]])
def test_the_largest_vocabulary(cuda_dev, draft, nodes):
    c, want = settled(lambda rng: make(nodes, 2000000, "bf16", draft, "chain", rng))
    assert np.array_equal(run(cuda_dev, c, "bf16")[:sum(nodes)], want)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("nodes", [[6], [20, 30, 4], [3] * 50])
def test_stars_of_likely_tokens(cuda_dev, draft, nodes):
    """Many children are turned down one after another: what is left gets small."""
    for seed in range(6):
        c, want = settled(lambda rng: make(nodes, 400, "f32", draft, "star",
                                           np.random.default_rng([seed, int(rng.integers(1 << 30))]), agree=1.0))
        c["u"] = np.maximum(c["u"], np.float32(0.9))
        picks, margin, drawn = wanted(c)
        if margin > 2e-5 and drawn > 1e-11:
            assert np.array_equal(run(cuda_dev, c, "f32"), picks)


@pytest.mark.parametrize("draft", [False, True])
def test_chains_without_parents_and_no_temperature(cuda_dev, draft):
    def one(rng):
        c = make([4, 7, 1], 3000, "bf16", draft, "chain", rng, heat=None)
        c["parents"] = None
        return c
    c, want = settled(one)
    assert np.array_equal(run(cuda_dev, c, "bf16"), want)
    st = torch.cuda.Stream(cuda_dev)
    torch.cuda.synchronize()
    assert np.array_equal(run(cuda_dev, c, "bf16", stream=st), want)


@pytest.mark.parametrize("many", [1, 40])
def test_rows_with_masks_infinities_and_nan(cuda_dev, many):
    """One request of each kind, alone (a cluster per node) and among others (per request)."""
    V = 777
    rng = np.random.default_rng(3)
    kinds = ["masked", "one", "none", "inf", "nan", "low", "cold", "hot", "equal"] * many
    c = make([3] * len(kinds), V, "f32", False, "chain", rng, heat=(1.0,))
    for b, kind in enumerate(kinds):
        row = c["x"][3 * b]
        if kind == "masked":
            row[rng.random(V) < 0.99] = -np.inf
        elif kind == "one":
            row[:] = -np.inf
            row[5] = -3
        elif kind == "none":
            row[:] = -np.inf
        elif kind == "inf":
            row[[9, 500]] = np.inf
        elif kind == "nan":
            row[::2] = np.nan
        elif kind == "low":
            row[rng.random(V) < 0.5] = np.finfo(np.float32).min
        elif kind == "cold":
            c["T"][b] = 1e-30
        elif kind == "hot":
            row[::3] = -np.inf
            c["T"][b] = np.inf
        elif kind == "equal":
            row[:] = 0.25
        good = np.nan_to_num(row, nan=-np.inf, posinf=np.inf, neginf=-np.inf)
        c["tokens"][3 * b + 1] = int(np.argmax(good)) if b % 2 else (int(np.argmax(good)) + 1) % V
    picks, margin, drawn = wanted(c)
    assert margin > 2e-5 and drawn > 1e-11
    assert np.array_equal(run(cuda_dev, c, "f32"), picks)
    assert (picks[0::3][[k == "none" for k in kinds]] == -1).all()


@pytest.mark.parametrize("many", [1, 60])
def test_residuals_with_nothing_left(cuda_dev, many):
    """Draft rows that leave nothing: the largest is taken, and the path goes on to a child
    that has it as its token, however the work is dealt."""
    V = 64
    x = np.zeros((4 * many, V), np.float32)
    x[:, 7] = 4.0
    one = np.array([0, 7, 9, 3])
    c = dict(x=x, cu=(4 * np.arange(many + 1)).tolist(), parents=[-1, 0, 0, 1] * many, tokens=np.tile(one, many),
             u=np.full(4 * many, 0.9, np.float32), d=np.full(many, 0.5, np.float32), T=None,
             q=np.full((4 * many, V), 2.0, np.float32))
    picks, _, _ = wanted(c)
    assert picks[:4].tolist() == [7, 7, -1, -1]
    assert np.array_equal(run(cuda_dev, c, "f32"), picks)


def test_requests_left_out_and_bad_parents(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    for many in (1, 50):  # a cluster per node, and per request
        nodes = [3, 2, 4] * many
        c, want = settled(lambda rng: make(nodes, 500, "f32", False, "mixed", rng))
        args = [i32(c["cu"], cuda_dev), i32(c["parents"], cuda_dev), i32(c["tokens"], cuda_dev),
                f32(c["u"], cuda_dev), f32(c["d"], cuda_dev)]
        x, T = f32(c["x"], cuda_dev), f32(c["T"], cuda_dev)
        out = paged.verify_picks(x, *args, max_nodes=3, temperature=T).cpu().numpy()  # 4 nodes are too many
        assert _lib.device_error(clear=True)[0] == _lib.ERR_POSITION
        for b, k in enumerate(nodes):
            at = slice(c["cu"][b], c["cu"][b + 1])
            assert np.array_equal(out[at], want[at] if k < 4 else [-1] * 4)
        args[1][1] = 2  # a parent behind its child: nobody's child
        paged.verify_picks(x, *args, max_nodes=4, temperature=T)
        assert _lib.device_error(clear=True) == (_lib.ERR_POSITION, 0)


def test_draws_at_their_ends_and_replay(cuda_dev):
    """Numbers 0 and just under 1; a captured call reads new numbers at its replay."""
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    rng = np.random.default_rng(0)
    V, B = 4099, 8
    c = make([1] * B, V, "f16", False, "chain", rng, heat=(1.0,))
    for b in range(B):
        c["x"][b, [b, V - 1 - b]] = 0.0
        c["x"][b, :b] = -np.inf
        c["x"][b, V - b:] = -np.inf
    c["d"][:] = [0.0, 1 - 2.0 ** -24] * (B // 2)
    picks = run(cuda_dev, c, "f16")
    assert np.array_equal(picks, [b if b % 2 == 0 else V - 1 - b for b in range(B)])
    x, T = torch.from_numpy(c["x"]).to(cuda_dev).half(), f32(c["T"], cuda_dev)
    args = [i32(c["cu"], cuda_dev), i32(c["parents"], cuda_dev), i32(c["tokens"], cuda_dev), f32(c["u"], cuda_dev),
            f32(c["d"], cuda_dev)]
    out = torch.empty(B, dtype=torch.int32, device=cuda_dev)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        paged.verify_picks(x, *args, max_nodes=1, temperature=T, out=out)
    for seed in range(3):
        c["d"] = np.random.default_rng(seed).random(B).astype(np.float32)
        args[-1].copy_(f32(c["d"], cuda_dev))
        g.replay()
        torch.cuda.synchronize()
        want, _, drawn = wanted(c)
        assert drawn > 1e-11 and np.array_equal(out.cpu().numpy(), want)
    _lib.raise_device_error()


def test_sampled_tokens_have_the_models_distribution(cuda_dev):
    """What stands after node 0 over 20,000 requests of the same logits, drafted by rows
    and certain: each of 12 tokens within 5 standard deviations of its probability."""
    rng = np.random.default_rng(5)
    V, B = 12, 20000
    x = (1.5 * rng.standard_normal(V)).astype(np.float32)
    p = np.exp(x.astype(np.float64))
    p /= p.sum()
    y = np.exp(x + rng.standard_normal(V))
    q = (y / y.sum()).astype(np.float32)
    for draft in (True, False):
        kids = rng.choice(V, (B, 2), p=q.astype(np.float64) / q.sum(dtype=np.float64)) if draft else np.tile([3, 8], (B, 1))
        c = dict(x=np.tile(x, (3 * B, 1)), cu=(3 * np.arange(B + 1)).tolist(), parents=[-1, 0, 0] * B,
                 tokens=np.concatenate([np.zeros((B, 1), int), kids], 1).ravel(), u=rng.random(3 * B).astype(np.float32),
                 d=rng.random(B).astype(np.float32), T=None, q=np.tile(q, (3 * B, 1)) if draft else None)
        first = run(cuda_dev, c, "f32", max_nodes=3)[::3]
        seen = np.bincount(first, minlength=V) / B
        assert (np.abs(seen - p) < 5 * np.sqrt(p * (1 - p) / B)).all(), (seen, p)


def test_refusals(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib, paged
    x = torch.zeros((3, 64), device=cuda_dev)
    cu, tok, par = i32([0, 3], cuda_dev), i32([0, 1, 2], cuda_dev), i32([-1, 0, 1], cuda_dev)
    u, d = f32([0.1, 0.2, 0.3], cuda_dev), f32([0.5], cuda_dev)
    assert paged.verify_picks(x, cu, par, tok, u, d, max_nodes=3).shape == (3,)
    assert paged.verify_picks(x[:0], i32([0, 0], cuda_dev), par[:0], tok[:0], u[:0], d, max_nodes=3).shape == (0,)
    for args, kw in (((x.cpu(), cu, par, tok, u, d), {}), ((x.t(), cu, par, tok, u, d), {}),
                     ((x.double(), cu, par, tok, u, d), {}), ((x, cu.long(), par, tok, u, d), {}),
                     ((x, cu, par[:2], tok, u, d), {}), ((x, cu, par, tok[:2], u, d), {}),
                     ((x, cu, par, tok, u[:2], d), {}), ((x, cu, par, tok, u.double(), d), {}),
                     ((x, cu, par, tok, u, d[:0]), {}), ((x, cu, par, tok, u, d), dict(max_nodes=0)),
                     ((x, cu, par, tok, u, d), dict(max_nodes=129)),
                     ((x, cu, par, tok, u, d), dict(temperature=f32([1, 1], cuda_dev))),
                     ((x, cu, par, tok, u, d), dict(draft=x[:2])), ((x, cu, par, tok, u, d), dict(draft=x.half())),
                     ((x, cu, par, tok, u, d), dict(out=tok.long()))):
        with pytest.raises((_lib.B2AError, KeyError)):
            paged.verify_picks(*args, **{"max_nodes": 3, **kw})
