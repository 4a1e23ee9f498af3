"""DraftStep at its limits: what its kernels would leave out is refused on the
host, before anything is launched or any page taken."""
import numpy as np
import pytest

from tests.conftest import rel_err
from tests.golden import cases

pytestmark = pytest.mark.gpu


def make(dev, **kw):
    from alpacca_open_sourced_by_jt_b200.decode_chain import LlamaQ8
    from alpacca_open_sourced_by_jt_b200.draft_step import DraftStep
    return DraftStep(LlamaQ8.from_spec(cases.llama_q8_case(), dev), **kw)


@pytest.mark.parametrize("max_len,page", [(100, 64), (100, 16), (128, 64)])
def test_rows_past_max_len_are_refused(cuda_dev, max_len, page):
    """The table's last page may hold rows past max_len; the step may not."""
    from alpacca_open_sourced_by_jt_b200 import _lib
    rng = np.random.default_rng(page)
    s = make(cuda_dev, requests=2, n_pages=32, page_rows=page, max_len=max_len)
    ids = rng.integers(0, s.m.V, max_len + 10).tolist()
    with pytest.raises(_lib.B2AShapeError):
        s.prefill([ids[:max_len + 1], ids[:3]])
    assert s.lens.tolist() == [0, 0] and s.ring_state.tolist() == [0, 32]
    first = s.prefill([ids[:max_len - 2], ids[:max_len]])
    assert min(first) >= 0 and s.lens.tolist() == [max_len - 2, max_len]
    with pytest.raises(_lib.B2AShapeError):
        s.verify([([first[0], 1, 2], [-1, 0, 0]), None])  # rows max_len - 2 .. max_len
    with pytest.raises(_lib.B2AShapeError):
        s.verify([None, ([first[1]], [-1])])
    # up to the limit the logits are those of a step with room to spare, within the
    # bar of test_draft_step_gpu.py (the residual GEMMs' sums have no fixed order)
    wide = make(cuda_dev, requests=2, n_pages=32, page_rows=page, max_len=512)
    wide.prefill([ids[:max_len - 2], ids[:max_len]])
    tree = [([first[0], 1], [-1, 0]), None]
    new = s.verify(tree)
    wide.verify(tree)
    assert rel_err(s.logits.cpu().numpy(), wide.logits.cpu().numpy()) < 2e-2
    assert min(new[0]) >= 0 and new[1] is None and s.lens.tolist() == [max_len - 2 + len(new[0]), max_len]
    s.end([0, 1])
    assert s.prefill([[], ids[:max_len]])[1] >= 0  # the place of an ended request starts at 0
    assert s.lens.tolist() == [0, max_len]
    _lib.raise_device_error()


def test_tokens_parents_and_counts_are_refused(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib
    s = make(cuda_dev, requests=2, n_pages=32, page_rows=16, max_len=400)
    V = s.m.V
    for prompts in ([[1, V], []], [[-1], []], [[1]], [[1], [2], [3]]):
        with pytest.raises(_lib.B2AShapeError):
            s.prefill(prompts)
    s.prefill([[1, 2], [3]])
    free = s.ring_state.tolist()
    for tree in (([V], [-1]), ([1, -1], [-1, 0]), ([1, 2], [-1, 1]), ([1, 2], [-1, -2]), ([1, 2], [-1]),
                 ([], []), ([1] * 129, [-1] + [0] * 128)):
        with pytest.raises(_lib.B2AShapeError):
            s.verify([tree, None])
    assert s.ring_state.tolist() == free and s.lens.tolist() == [2, 1]
    assert len(s.verify([([1] * 128, [-1] + [0] * 127), ([4], [-1])])) == 2
    _lib.raise_device_error()


def test_step_of_no_trees(cuda_dev):
    from alpacca_open_sourced_by_jt_b200 import _lib
    s = make(cuda_dev, requests=2, n_pages=8, page_rows=16, max_len=64)
    assert s.verify([None, None]) == [None, None] and s.prefill([[], []]) == [-1, -1]
    first = s.prefill([[5, 6], []])
    assert s.verify([None, None]) == [None, None] and s.lens.tolist() == [2, 0]
    assert len(s.verify([([first[0]], [-1]), None])[0]) == 1
    _lib.raise_device_error()
