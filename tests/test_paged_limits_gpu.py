"""The paged-cache and draft-tree operators at their limits: padded steps,
requests that find no pages, that end or are out of bounds, numbers that are not
finite where nothing may see them.  Definitions in paged_ref.py; bookkeeping is
equal, attention within the bounds that test_paged_gpu.py derives."""
import numpy as np
import pytest
import torch

from tests import paged_ref as ref

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
