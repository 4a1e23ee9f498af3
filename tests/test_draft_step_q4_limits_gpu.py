"""DraftStep's sampled steps: what they read (test_draft_step_q4_gpu.py has the forward
pass)."""
import numpy as np
import pytest
import torch

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
