"""DraftStep (draft_step.py) against the one-sequence chains of the same model:
logits of every accepted token within 2e-2 of DecodeChain's (the bar of the
prefill chunks, which run the same 16-bit GEMMs), the committed K rows within
2e-2 absolute, and the greedy continuation the same whatever is drafted, as far
as its picks lead by more than that bar (two tokens closer than the rounding of
16-bit operands may change places)."""
import numpy as np
import pytest
import torch

from tests.conftest import max_abs_err, rel_err
from tests.golden import cases

pytestmark = pytest.mark.gpu


def _model(dev):
    from alpacca_open_sourced_by_jt_b200.decode_chain import LlamaQ8
    return LlamaQ8.from_spec(cases.llama_q8_case(), dev)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 64])
def test_verified_trees_follow_the_model(cuda_dev, dt, page):
    from alpacca_open_sourced_by_jt_b200 import _lib
    from alpacca_open_sourced_by_jt_b200.decode_chain import DecodeChain
    from alpacca_open_sourced_by_jt_b200.draft_step import DraftStep
    model = _model(cuda_dev)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, model.V, n).tolist() for n in (5, 150, 1)]

    def greedy(drafts):
        """12 tokens or more per request; drafts(b, known) -> a list of chains to
        try behind the request's last token."""
        s = DraftStep(model, 3, 24, page_rows=page, max_len=512, dtype=dt)
        out = [[t] for t in s.prefill(prompts)]
        steps, sure = 0, [1, 1, 1]  # tokens picked by more than the bar
        while min(len(o) for o in out) < 12:
            trees = []
            for b in range(3):
                tokens, parents = [out[b][-1]], [-1]
                for chain in drafts(b, out[b]):
                    up = 0
                    for t in chain:
                        tokens.append(t)
                        parents.append(up)
                        up = len(tokens) - 1
                trees.append((tokens, parents))
            for b, new in enumerate(s.verify(trees)):
                if s.logits.shape[0] == 3 and sure[b] == len(out[b]):
                    top = s.logits[b].topk(2).values
                    sure[b] += int(top[0] - top[1] > 2e-2 * s.logits[b].abs().max())
                out[b] += new
            steps += 1
        _lib.raise_device_error()
        return s, out, steps, sure

    _, plain, steps0, sure = greedy(lambda b, known: [])
    # drafts: a wrong chain first, then the right continuation with a wrong end
    right = lambda b, known: [[1, 2], plain[b][len(known):len(known) + 3] + [7]]  # noqa: E731
    s, out, steps1, _ = greedy(right)
    for b in range(3):
        n = min(len(out[b]), sure[b])
        assert out[b][:n] == plain[b][:n]
    assert steps1 < steps0  # the drafts were accepted
    for b in range(3):
        chain = DecodeChain(model, 512, dt)
        seq = prompts[b] + out[b]
        n = int(s.lens[b])
        for i in range(n):
            logits = chain(seq[i], i).numpy().copy()
        t = s.table[b].long()
        rows = torch.arange(n, device=cuda_dev)
        k = s.k_pool[:, t[rows // page], rows % page]
        for li in range(len(model.layers)):
            assert max_abs_err(k[li].float().cpu().numpy(),
                               chain.k_cache[li][0, :n].float().cpu().numpy()) < 2e-2
        # the chain's logits after the last cached token pick the token that follows
        assert logits[out[b][n - len(prompts[b])]] >= logits.max() - 2e-2 * np.abs(logits).max()


def test_logits_of_a_tree_match_the_chain(cuda_dev):
    from alpacca_open_sourced_by_jt_b200.decode_chain import DecodeChain
    from alpacca_open_sourced_by_jt_b200.draft_step import DraftStep
    model = _model(cuda_dev)
    s = DraftStep(model, 1, 8, page_rows=16, max_len=128)
    prompt = [3, 1, 4, 1, 5]
    s.prefill([prompt])
    tokens, parents = [9, 2, 6, 5, 3], [-1, 0, 0, 1, 2]
    s.verify([(tokens, parents)])
    for i in range(5):
        path, at = [], i
        while at >= 0:
            path.append(tokens[at])
            at = parents[at]
        chain = DecodeChain(model, 128, torch.float16)
        for p, t in enumerate(prompt + path[::-1]):
            logits = chain(t, p).numpy().copy()
        assert rel_err(s.logits[i].cpu().numpy(), logits) < 2e-2


def test_penalties_pages_and_refusals(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib
    from alpacca_open_sourced_by_jt_b200.draft_step import DraftStep
    model = _model(cuda_dev)
    with pytest.raises(_lib.B2AShapeError):
        DraftStep(model, 1, 4, dtype=torch.float32)
    s = DraftStep(model, 2, 4, page_rows=16, max_len=128)
    first = s.prefill([[3, 1, 4], []])
    assert first[1] == -1 and s.lens.tolist() == [3, 0]
    # a mask that allows one token only
    mask = torch.zeros((1, model.V // 32), dtype=torch.int32, device=cuda_dev)
    mask[0, 5] = 1 << 3
    assert s.verify([([first[0]], [-1]), None], mask=mask) == [[5 * 32 + 3], None]
    assert s.lens.tolist() == [4, 0] and s.ring_state[1].item() == 3
    with pytest.raises(_lib.B2AError):
        s.prefill([[], list(range(100))])  # 7 pages, 3 are free
    s.end([0])
    assert s.ring_state[1].item() == 4 and s.lens.tolist() == [0, 0]
    assert s.prefill([[], list(range(64))])[1] >= 0
