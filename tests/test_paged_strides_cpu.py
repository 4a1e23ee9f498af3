"""Broadcast (expanded) tensors have a stride of 0, which means "dense" to the C calls: they
would read, or write, behind the one row or page that is there.  The wrappers refuse them,
before anything is launched: with tensors that have a device, shapes and strides but no
memory."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from alpacca_open_sourced_by_jt_b200 import _lib, paged

H, KV, D, page, pages, n, B = 8, 2, 64, 16, 4, 3, 1


@pytest.fixture
def made():
    with FakeTensorMode():
        i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
        f16 = lambda *s: torch.empty(s, dtype=torch.float16, device="cuda")  # noqa: E731
        yield dict(q=f16(n, H, D), one_q=f16(1, H, D).expand(n, H, D), k=f16(n, KV, D), i32=i32,
                   pool=torch.empty((pages, KV, page // 16, 18 * D), dtype=torch.uint8, device="cuda"),
                   one_page=torch.empty((1, KV, page // 16, 18 * D), dtype=torch.uint8, device="cuda").expand(pages, -1, -1, -1),
                   kp=f16(pages, page, KV, D), one_kp=f16(1, page, KV, D).expand(pages, -1, -1, -1),
                   tab=torch.empty((8, D // 2), device="cuda"))


def refused(call, *args, **kw):
    with pytest.raises(_lib.B2AShapeError):
        call(*args, **kw)


def test_rows_of_q(made):
    tree = (made["i32"](B), made["i32"](B + 1), made["i32"](n))
    kw = dict(table=made["i32"](B, pages), max_nodes=n)
    refused(paged.tree_decode_q4, made["one_q"], made["pool"], *tree, **kw)
    refused(paged.tree_decode, made["one_q"], made["kp"], made["kp"], *tree, **kw)


def test_pages(made):
    m = made
    tree = (m["i32"](B), m["i32"](B + 1), m["i32"](n))
    kw = dict(table=m["i32"](B, pages), max_nodes=n)
    refused(paged.tree_decode_q4, m["q"], m["one_page"], *tree, **kw)
    refused(paged.q4_rows, m["one_page"], m["i32"](n))
    rows = (m["q"], m["k"], m["k"], m["i32"](n), m["i32"](n), m["tab"], m["tab"])
    refused(paged.rope_append_q4, *rows, pool=m["one_page"])
    refused(paged.tree_commit_q4, m["i32"](n), m["i32"](n), m["i32"](n), tree[1], tree[0], m["one_page"], **kw)
    refused(paged.tree_decode, m["q"], m["one_kp"], m["one_kp"], *tree, **kw)
    refused(paged.rope_append, *rows, k_pool=m["one_kp"], v_pool=m["one_kp"])
    refused(paged.tree_commit, m["i32"](n), m["i32"](n), m["i32"](n), tree[1], tree[0], m["one_kp"], m["one_kp"], **kw)


def test_overlapping_pages(made):
    base = torch.empty(10000, dtype=torch.uint8, device="cuda")
    shape = (pages, KV, page // 16, 18 * D)
    strides = (18 * D, 18 * D * page // 16, 18 * D, 1)  # pages one head apart
    refused(paged.q4_rows, base.as_strided(shape, strides), made["i32"](n))
