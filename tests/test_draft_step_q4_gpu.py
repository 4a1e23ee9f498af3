"""DraftStep with a 4-bit cache, with models that norm their heads, and sampling.

The forward pass is restated in 64 bits over the rows that the step's own cache holds:
logits within 2e-2 (the bar of test_draft_step_gpu.py: the same 16-bit GEMMs).  The
cached rows themselves: each within half a step of its block's scale (a whole one at the
end of the range without a code) of the restated K and V, and 2e-2 of the largest for the
GEMMs.  Sampled picks are equal to the definition's on the step's own logits."""
import math

import numpy as np
import pytest
import torch

from oracle.llama_q8 import q8_0_row, q8_0_unpack
from tests import paged_ref as ref
from tests import q4_ref
from tests.conftest import rel_err
from tests.golden import cases

pytestmark = pytest.mark.gpu


def spec_of(kind):
    spec = cases.llama_q8_case()
    if kind == "norm":
        return spec
    rng = np.random.default_rng(17)
    norm = lambda: (1 + 0.2 * rng.standard_normal(spec["head_dim"])).astype(np.float32)  # noqa: E731
    return dict(spec, rope_style="neox", layers=[dict(ly, q_norm=norm(), k_norm=norm()) for ly in spec["layers"]])


def make(dev, kind, **kw):
    from alpacca_open_sourced_by_jt_b200.decode_chain import LlamaQ8
    from alpacca_open_sourced_by_jt_b200.draft_step import DraftStep
    return DraftStep(LlamaQ8.from_spec(spec_of(kind), dev), **kw)


def matrix(data, rows, cols):
    codes, d = q8_0_unpack(data, rows, cols)
    return codes.astype(np.float64) * np.repeat(d.astype(np.float64), 32, 1)


def plain(spec, seq, held_k, held_v):
    """Logits after seq's last token, K and V of every layer; attention reads the rows
    held_k, held_v (layers, n, KV, D)."""
    E, H, KV, D, F, V = (spec[k] for k in ("n_embd", "n_head", "n_kv", "head_dim", "n_ff", "n_vocab"))
    eps, n, style = spec["rms_eps"], len(seq), spec.get("rope_style", "norm")
    theta = np.outer(np.arange(n), spec["rope_base"] ** (-np.arange(0, D, 2) / D))
    norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w  # noqa: E731
    x = np.stack([q8_0_row(spec["tok_embd"], V, E, t) for t in seq]).astype(np.float64)
    ks, vs = [], []
    for li, ly in enumerate(spec["layers"]):
        h = norm(x, ly["attn_norm"])
        q = (h @ matrix(ly["wq"], H * D, E).T).reshape(n, H, D)
        k = (h @ matrix(ly["wk"], KV * D, E).T).reshape(n, KV, D)
        vs.append((h @ matrix(ly["wv"], KV * D, E).T).reshape(n, KV, D))
        turn = (np.cos(theta), np.sin(theta), D, style)
        q = q4_ref.heads64(q, ly.get("q_norm"), eps, *turn)
        ks.append(q4_ref.heads64(k, ly.get("k_norm"), eps, *turn))
        att = np.zeros((n, H, D))
        for g in range(H):
            s = q[:, g] @ held_k[li][:, g // (H // KV)].T / math.sqrt(D)
            s[np.triu_indices(n, 1)] = -np.inf
            p = np.exp(s - s.max(-1, keepdims=True))
            att[:, g] = p / p.sum(-1, keepdims=True) @ held_v[li][:, g // (H // KV)]
        x = x + att.reshape(n, -1) @ matrix(ly["wo"], E, H * D).T
        h = norm(x, ly["ffn_norm"])
        gate, up = h @ matrix(ly["w_gate"], F, E).T, h @ matrix(ly["w_up"], F, E).T
        x = x + (gate / (1 + np.exp(-gate)) * up) @ matrix(ly["w_down"], E, F).T
    return norm(x[-1], spec["out_norm"]) @ matrix(spec["output"], V, E).T, np.stack(ks), np.stack(vs)


def cached(s, b):
    """K and V rows (layers, n, KV, D) of request b, float64."""
    from alpacca_open_sourced_by_jt_b200 import paged
    r = torch.arange(int(s.lens[b]), device=s.table.device)
    pages = s.table[b][r // s.page_rows].long()
    if s.pool is None:
        return [x[:, pages, r % s.page_rows].double().cpu().numpy() for x in (s.k_pool, s.v_pool)]
    slots = (pages * s.page_rows + r % s.page_rows).int()
    rows = [paged.q4_rows(x, slots) for x in s.pool]
    return [torch.stack([kv[i] for kv in rows]).double().cpu().numpy() for i in (0, 1)]


def check_request(s, spec, b, seq, logits):
    k, v = cached(s, b)
    want, pk, pv = plain(spec, seq, k, v)
    assert rel_err(logits.cpu().numpy(), want.astype(np.float32)) < 2e-2
    for held, x in ((k, pk), (v, pv)):
        room = np.zeros_like(x)
        if s.pool is not None:
            blocks = x.reshape(*x.shape[:-1], -1, 32)
            m = np.abs(blocks).max(-1, keepdims=True)
            top = np.where(blocks.max(-1, keepdims=True) > -blocks.min(-1, keepdims=True), -1.0, 1.0) * blocks
            step = m / 8 * (1 + 2.0 ** -8)
            # code 0 stands for the value of largest magnitude, there is none for its opposite
            room = (np.where(top > 6.5 * m / 8, 1.0, 0.5) * step).reshape(x.shape)
            # (two largest values of opposite sign may change places)
            near = np.abs(np.abs(blocks.max(-1)) - np.abs(blocks.min(-1))) < 4e-2 * m[..., 0]
            room = np.where(np.repeat(near, 32, -1).reshape(x.shape), np.repeat(step, 32, -1).reshape(x.shape), room)
        assert (np.abs(held - x) <= room + 2e-2 * np.abs(x).max()).all()


@pytest.mark.parametrize("kind,kv_bits", [("norm", 4), ("neox, normed", 4), ("neox, normed", 16)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_steps_follow_the_model(cuda_dev, kind, kv_bits, dt):
    """Prompts, then greedy steps over trees and steps with sampled tokens."""
    from alpacca_open_sourced_by_jt_b200 import _lib
    rng = np.random.default_rng(1)
    spec = spec_of(kind)
    s = make(cuda_dev, kind, requests=3, n_pages=24, page_rows=32, max_len=400, dtype=dt, kv_bits=kv_bits)
    V = s.m.V
    seqs = [rng.integers(0, V, n).tolist() for n in (5, 170, 33)]
    last = s.prefill(seqs)
    taken = 0
    for step in range(6):
        sampled = step >= 2
        trees, drafts = [], []
        for b in range(3):
            n = int(rng.integers(1, 12)) if step else 1
            par = ref.random_tree(n, rng)
            # tokens that the model may well take: what it took last, or likely ones of the last logits
            tok = [last[b]] + [int(t) for t in rng.integers(0, V, n - 1)]
            if step and n > 1:
                likely = s.logits[-1].topk(4).indices.tolist()
                tok[1:] = [int(rng.choice(likely)) for _ in tok[1:]]
            trees.append((tok, par))
        cu = np.concatenate([[0], np.cumsum([len(t[0]) for t in trees])]).tolist()
        n = cu[-1]
        kw = {}
        if sampled:
            kw = dict(uniforms=torch.rand(n, device=cuda_dev), draws=torch.rand(3, device=cuda_dev))
            if step % 2:
                kw["temperature"] = torch.tensor([0.3, 0.0, 1.5], device=cuda_dev)
            if step > 3:
                kw["draft"] = torch.softmax(torch.randn((n, V), device=cuda_dev), -1)
        new = s.verify(trees, **kw)
        _lib.raise_device_error()
        host = {k: v.cpu().numpy() for k, v in kw.items()}
        tokens, parents = sum((t[0] for t in trees), []), sum((t[1] for t in trees), [])
        x = s.logits.float().cpu().numpy()
        if sampled:
            picks, margin, drawn = q4_ref.verify(x, cu, parents, np.array(tokens), host["uniforms"], host["draws"],
                                                 host.get("temperature"), host.get("draft"))
            if margin > 2e-5 and drawn > 1e-11:
                assert np.array_equal(s.picks.cpu().numpy(), picks)
        for b, (path, nxt) in enumerate(ref.accept(s.picks.tolist(), tokens, parents, cu)):
            assert new[b] == [trees[b][0][i] for i in path[1:]] + [nxt]
            seqs[b] += [trees[b][0][i] for i in path]
            last[b] = nxt
            taken += len(path) - 1
            assert int(s.lens[b]) == len(seqs[b])
            check_request(s, spec, b, seqs[b], s.logits[cu[b] + path[-1]])
    s.end([0, 2])
    _lib.raise_device_error()


def test_a_cache_of_4_bits_takes_its_bytes(cuda_dev):
    """18 bytes for 32 values."""
    s = make(cuda_dev, "norm", requests=1, n_pages=8, page_rows=16, max_len=64, kv_bits=4)
    wide = make(cuda_dev, "norm", requests=1, n_pages=8, page_rows=16, max_len=64)
    assert s.pool.numel() * 64 == (wide.k_pool.numel() + wide.v_pool.numel()) * 2 * 18 and s.k_pool is None


def test_certain_drafts_at_temperature_0_are_greedy(cuda_dev):
    """Sampling at temperature 0 gives what greedy verification gives."""
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, 1024, n).tolist() for n in (20, 70)]
    got = []
    for sampled in (False, True):
        s = make(cuda_dev, "neox, normed", requests=2, n_pages=24, page_rows=16, max_len=150, kv_bits=4)
        last = s.prefill(prompts)
        logits = []
        for _ in range(4):
            trees = [([t, 3, t], [-1, 0, 0]) for t in last]
            kw = dict(uniforms=torch.rand(6, device=cuda_dev), draws=torch.rand(2, device=cuda_dev),
                      temperature=torch.zeros(2, device=cuda_dev)) if sampled else {}
            new = s.verify(trees, **kw)
            top = s.logits.topk(2).values
            logits.append(bool((top[:, 0] - top[:, 1] > 2e-2 * s.logits.abs().amax(1)).all()))
            got.append((sampled, new))
            last = [t[-1] for t in new]
    n = 0
    while n < 4 and logits[n]:  # (sums in the GEMMs' epilogues have no fixed order)
        assert got[n][1] == got[4 + n][1]
        n += 1


def test_refusals(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib
    from alpacca_open_sourced_by_jt_b200.decode_chain import DecodeChain, LlamaQ8
    Bad = _lib.B2AShapeError
    with pytest.raises(Bad):
        make(cuda_dev, "norm", requests=1, n_pages=8, kv_bits=8)
    with pytest.raises(Bad):
        make(cuda_dev, "norm", requests=1, n_pages=8, page_rows=24, kv_bits=4)
    spec = spec_of("neox, normed")
    with pytest.raises(Bad):
        DecodeChain(LlamaQ8.from_spec(spec, cuda_dev), 64)
    with pytest.raises(Bad):
        LlamaQ8.from_spec(dict(spec, rope_style="gptj"), cuda_dev)
    with pytest.raises(Bad):
        LlamaQ8.from_spec(dict(spec, layers=[spec["layers"][0], spec_of("norm")["layers"][1]]), cuda_dev)
    with pytest.raises(Bad):
        LlamaQ8.from_spec(dict(spec, layers=[dict(ly, k_norm=ly["k_norm"][:32]) for ly in spec["layers"]]), cuda_dev)
    s = make(cuda_dev, "norm", requests=2, n_pages=8, page_rows=16, max_len=64, kv_bits=4)
    last = s.prefill([[1, 2, 3], [4]])
    state = (s.ring_state.tolist(), s.lens.tolist())
    u, d = torch.rand(3, device=cuda_dev), torch.rand(2, device=cuda_dev)
    trees = [([last[0], 5], [-1, 0]), ([last[1]], [-1])]
    for kw in (dict(uniforms=u), dict(draws=d), dict(temperature=d), dict(draft=torch.rand((3, s.m.V), device=cuda_dev)),
               dict(uniforms=u[:2], draws=d), dict(uniforms=u, draws=u), dict(uniforms=u.double(), draws=d),
               dict(uniforms=u, draws=d, temperature=u), dict(uniforms=u, draws=d, draft=torch.rand((3, 5), device=cuda_dev)),
               dict(uniforms=u, draws=d, draft=torch.rand((3, s.m.V), device=cuda_dev).half()),
               dict(uniforms=u.cpu(), draws=d)):
        with pytest.raises(_lib.B2AError):
            s.verify(trees, **kw)
    assert state == (s.ring_state.tolist(), s.lens.tolist())
    assert len(s.verify(trees, uniforms=u, draws=d)) == 2
    _lib.raise_device_error()
