"""DraftStep's sampled steps: what they read, and their picks counted request by request
(those whose decisions are clear; test_draft_step_q4_gpu.py has the forward pass)."""
import numpy as np
import pytest
import torch

from tests import paged_ref as ref
from tests import q4_ref
from tests.test_draft_step_q4_gpu import make

pytestmark = pytest.mark.gpu


def numbers(dev, n, requests, seed):
    g = torch.Generator().manual_seed(seed)
    return dict(uniforms=torch.rand(n, generator=g).to(dev), draws=torch.rand(requests, generator=g).to(dev))


def test_sampled_steps_read_the_rows_on_their_paths_only(cuda_dev, monkeypatch):
    """Without limits there is nothing to be done to the logits, and the greedy picks of all
    rows are nobody's: verify_picks alone looks at the rows."""
    from alpacca_open_sourced_by_jt_b200 import paged
    calls = []
    plain = paged.constrain_logits
    monkeypatch.setattr(paged, "constrain_logits", lambda *a, **k: calls.append(k) or plain(*a, **k))
    s = make(cuda_dev, "norm", requests=2, n_pages=16, page_rows=16, max_len=100, kv_bits=4)
    last = s.prefill([[1, 2, 3], [4, 5]])
    trees = [([last[0], 5, 6], [-1, 0, 0]), ([last[1], 9], [-1, 0])]
    del calls[:]
    new = s.verify(trees, **numbers(cuda_dev, 5, 2, 0))
    assert not calls
    picks, _, _ = q4_ref.verify(s.logits.cpu().numpy(), [0, 3, 5], [-1, 0, 0, -1, 0],
                                np.array([last[0], 5, 6, last[1], 9]), *(x.cpu().numpy() for x in numbers(cuda_dev, 5, 2, 0).values()),
                                None, None)
    assert np.array_equal(s.picks.cpu().numpy(), picks)
    # limits count, sampled or not; a mask that leaves one token leaves no choice
    mask = torch.zeros((2, -(-s.m.V // 32)), dtype=torch.int32, device=cuda_dev)
    mask[:, 1] = 1 << 3
    got = s.verify([([t[-1]], [-1]) for t in new], **numbers(cuda_dev, 2, 2, 1), mask=mask)
    assert len(calls) == 1 and got == [[35], [35]]
    s.verify([([t[-1]], [-1]) for t in got])
    assert len(calls) == 2


def test_a_broadcast_draft_is_refused_before_the_step_takes_pages(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib
    s = make(cuda_dev, "norm", requests=1, n_pages=8, page_rows=16, max_len=64, kv_bits=4)
    last = s.prefill([list(range(15))])
    state = (s.ring_state.tolist(), s.held.tolist(), s.lens.tolist())
    tree = ([last[0], 5, 6], [-1, 0, 0])  # (its rows begin a page)
    row = torch.full((1, s.m.V), 1 / s.m.V, device=cuda_dev)
    with pytest.raises(_lib.B2AShapeError):
        s.verify([tree], **numbers(cuda_dev, 3, 1, 0), draft=row.expand(3, -1))
    assert state == (s.ring_state.tolist(), s.held.tolist(), s.lens.tolist())
    assert len(s.verify([tree], **numbers(cuda_dev, 3, 1, 0), draft=row.repeat(3, 1))) == 1


@pytest.mark.parametrize("kv_bits", [4, 16])
def test_sampled_picks_are_the_definitions(cuda_dev, kv_bits):
    from alpacca_open_sourced_by_jt_b200 import _lib
    rng = np.random.default_rng(6)
    s = make(cuda_dev, "neox, normed", requests=3, n_pages=32, page_rows=16, max_len=300, kv_bits=kv_bits)
    last = s.prefill([rng.integers(0, s.m.V, n).tolist() for n in (5, 40, 17)])
    s.verify([([t], [-1]) for t in last])
    last = s.picks.tolist()
    compared = 0
    for step in range(8):
        trees = []
        likely = s.logits[-1].topk(4).indices.tolist()
        for t in last:
            n = int(rng.integers(1, 10))
            trees.append(([t] + [int(rng.choice(likely)) for _ in range(n - 1)], ref.random_tree(n, rng)))
        cu = np.concatenate([[0], np.cumsum([len(t[0]) for t in trees])]).tolist()
        kw = numbers(cuda_dev, cu[-1], 3, step)
        if step % 2:
            kw["temperature"] = torch.tensor([0.3, 0.8, 1.5], device=cuda_dev)
        if step > 4:
            kw["draft"] = torch.softmax(torch.randn((cu[-1], s.m.V), device=cuda_dev), -1)
        new = s.verify(trees, **kw)
        _lib.raise_device_error()
        last = [t[-1] for t in new]
        host = {k: v.cpu().numpy() for k, v in kw.items()}
        x, got = s.logits.cpu().numpy(), s.picks.cpu().numpy()
        for b, (tok, par) in enumerate(trees):
            at = slice(cu[b], cu[b + 1])
            picks, margin, drawn = q4_ref.verify(
                x[at], [0, len(tok)], par, np.array(tok), host["uniforms"][at], host["draws"][b:b + 1],
                host["temperature"][b:b + 1] if "temperature" in kw else None, host["draft"][at] if "draft" in kw else None)
            if margin > 2e-5 and drawn > 1e-11:
                assert np.array_equal(got[at], picks)
                compared += 1
    assert compared >= 20, compared


def test_temperature_0_is_greedy_wherever_the_logits_are_clear(cuda_dev):
    """Each step of both from the same rows: a request is followed as long as the rows on
    its path have one clear largest logit (the GEMMs' sums have no fixed order)."""
    compared = 0
    for seed in range(4):
        rng = np.random.default_rng(seed)
        prompts = [rng.integers(0, 1024, n).tolist() for n in (20, 70)]
        steps = [make(cuda_dev, "neox, normed", requests=2, n_pages=24, page_rows=16, max_len=150, kv_bits=4) for _ in (0, 1)]
        last = steps[0].prefill(prompts)
        steps[1].prefill(prompts)
        same = [True, True]
        for i in range(4):
            trees = [([t, 3, t], [-1, 0, 0]) for t in last]
            greedy = steps[0].verify(trees)
            sampled = steps[1].verify(trees, **numbers(cuda_dev, 6, 2, i), temperature=torch.zeros(2, device=cuda_dev))
            top = steps[0].logits.topk(2).values
            clear = (top[:, 0] - top[:, 1] > 2e-2 * steps[0].logits.abs().amax(1)).view(2, 3).all(1).tolist()
            for b in (0, 1):
                same[b] = same[b] and clear[b]
                if same[b]:
                    assert greedy[b] == sampled[b]
                    compared += 1
            if not any(same):
                break
            last = [t[-1] for t in greedy]
    assert compared >= 4, compared
