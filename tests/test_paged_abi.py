"""Host-side refusals of the paged-cache and draft-tree entries: every case
returns before any CUDA call (the addresses are never read)."""
import pytest

from alpacca_open_sourced_by_jt_b200 import _lib, build

P = 1 << 20
F16, F32 = _lib.F16, _lib.F32


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


CALLS = {
    "page_plan": dict(lens=P, add=P, parents=None, held=P, held_out=2 * P, table=P, stride=8, ring=P,
                      ring_size=64, state=P, state_out=2 * P, cu=P, seq=P, pos=P, slot=P, B=4,
                      max_tokens=16, max_pages=8, page_rows=16, stream=None),
    "rope_append_paged": dict(q=P, qs=512, k=P, ks=128, v=P, vs=128, dt=F32, bq=None, bk=None, bv=None,
                              cos=P, sin=P, tab_rows=16, pos=P, slot=P, kp=P, vp=P, n_pages=4,
                              page_rows=16, page_stride=0, kv_dt=F16, q_out=P, qo_dt=F16, n_tok=0, H=8,
                              KV=2, D=64, n_rot=64, style=0, stream=None),
    "tree_decode": dict(q=P, qs=0, k=P, v=P, n_pages=64, page_rows=16, page_stride=0, table=P, stride=8,
                        width=8, lens=P, cu=P, parents=P, out=P, lse=None, ws=P, ws_bytes=1 << 30, B=2,
                        n_tok=0, max_nodes=8, H=8, KV=2, D=64, dt=F16, scale=0.125, max_len=128,
                        stream=None),
    "constrain_logits": dict(x=P, xs=1000, dt=F32, out=2 * P, os=1000, odt=F32, picks=P, cu=P,
                             parents=None, tokens=None, hist=P, hist_start=P, n_hist=5, prompt=None,
                             rep=None, pres=None, freq=None, bstart=P, bids=P, bias=P, n_bias=3, mask=P,
                             ms=32, B=2, n_rows=0, max_nodes=4, V=1000, ws=P, ws_bytes=1 << 30,
                             stream=None),
    "tree_commit": dict(picks=P, tokens=P, parents=None, cu=P, lens=P, table=P, stride=8, width=8, k=P,
                        v=P, L=2, layer_stride=1 << 20, n_pages=64, page_rows=16, page_stride=0, KV=2,
                        D=64, dt=F16, B=2, n_tok=8, max_nodes=8, max_len=128, path=P, acc=P, next=P,
                        lens_out=2 * P, stream=None),
}


def call(lib, name, **kw):
    args = dict(CALLS[name])
    assert set(kw) <= set(args)
    args.update(kw)
    return getattr(lib, "b2a_" + name)(*args.values())


@pytest.mark.parametrize("name", ["rope_append_paged", "tree_decode", "constrain_logits"])
def test_no_tokens_is_a_successful_no_op(lib, name):
    assert call(lib, name) == _lib.OK


BAD = [
    ("page_plan", dict(lens=None), _lib.ERR_ARG),
    ("page_plan", dict(slot=None), _lib.ERR_ARG),
    ("page_plan", dict(B=0), _lib.ERR_ARG),
    ("page_plan", dict(B=4096), _lib.ERR_UNSUPPORTED),
    ("page_plan", dict(page_rows=24), _lib.ERR_SHAPE),
    ("page_plan", dict(stride=7), _lib.ERR_SHAPE),
    ("page_plan", dict(held_out=P), _lib.ERR_ARG),
    ("page_plan", dict(state_out=P), _lib.ERR_ARG),
    ("page_plan", dict(ring_size=1 << 28), _lib.ERR_UNSUPPORTED),
    ("rope_append_paged", dict(q=None), _lib.ERR_ARG),
    ("rope_append_paged", dict(n_tok=-1), _lib.ERR_ARG),
    ("rope_append_paged", dict(D=63), _lib.ERR_UNSUPPORTED),
    ("rope_append_paged", dict(D=512), _lib.ERR_UNSUPPORTED),
    ("rope_append_paged", dict(n_rot=66), _lib.ERR_SHAPE),
    ("rope_append_paged", dict(n_rot=31), _lib.ERR_SHAPE),
    ("rope_append_paged", dict(style=2), _lib.ERR_ARG),
    ("rope_append_paged", dict(dt=9), _lib.ERR_DTYPE),
    ("rope_append_paged", dict(page_rows=20), _lib.ERR_SHAPE),
    ("rope_append_paged", dict(page_stride=100), _lib.ERR_SHAPE),
    ("rope_append_paged", dict(ks=64), _lib.ERR_SHAPE),
    ("tree_decode", dict(cu=None), _lib.ERR_ARG),
    ("tree_decode", dict(max_nodes=0), _lib.ERR_ARG),
    ("tree_decode", dict(max_nodes=129), _lib.ERR_ARG),
    ("tree_decode", dict(H=9), _lib.ERR_SHAPE),
    ("tree_decode", dict(D=96), _lib.ERR_UNSUPPORTED),
    ("tree_decode", dict(dt=5), _lib.ERR_DTYPE),
    ("tree_decode", dict(scale=0.0), _lib.ERR_ARG),
    ("tree_decode", dict(scale=float("inf")), _lib.ERR_ARG),
    ("tree_decode", dict(page_rows=8), _lib.ERR_SHAPE),
    ("tree_decode", dict(page_rows=48), _lib.ERR_SHAPE),
    ("tree_decode", dict(max_len=129), _lib.ERR_SHAPE),
    ("tree_decode", dict(stride=4), _lib.ERR_SHAPE),
    ("tree_decode", dict(table=None, n_pages=1, page_rows=512), _lib.ERR_SHAPE),
    ("tree_decode", dict(table=None, page_rows=100), _lib.ERR_SHAPE),
    ("tree_decode", dict(page_stride=100), _lib.ERR_SHAPE),
    ("tree_decode", dict(qs=100), _lib.ERR_SHAPE),
    ("tree_decode", dict(qs=513), _lib.ERR_ALIGN),
    ("tree_decode", dict(q=P + 2), _lib.ERR_ALIGN),
    ("tree_decode", dict(H=400, KV=2, n_tok=1), _lib.ERR_UNSUPPORTED),
    ("tree_decode", dict(n_tok=4, ws_bytes=64, max_len=4096, width=256, stride=256), _lib.ERR_WORKSPACE),
    ("constrain_logits", dict(picks=None), _lib.ERR_ARG),
    ("constrain_logits", dict(V=0), _lib.ERR_ARG),
    ("constrain_logits", dict(max_nodes=200), _lib.ERR_ARG),
    ("constrain_logits", dict(B=70000), _lib.ERR_UNSUPPORTED),
    ("constrain_logits", dict(hist_start=None), _lib.ERR_ARG),
    ("constrain_logits", dict(bids=None), _lib.ERR_ARG),
    ("constrain_logits", dict(dt=4), _lib.ERR_DTYPE),
    ("constrain_logits", dict(xs=999), _lib.ERR_SHAPE),
    ("constrain_logits", dict(ms=31), _lib.ERR_SHAPE),
    ("constrain_logits", dict(out=P, odt=F16), _lib.ERR_ARG),
    ("constrain_logits", dict(n_rows=2, ws_bytes=8), _lib.ERR_WORKSPACE),
    ("constrain_logits", dict(n_rows=2, ws=P + 4), _lib.ERR_ALIGN),
    ("tree_commit", dict(path=None), _lib.ERR_ARG),
    ("tree_commit", dict(L=0), _lib.ERR_ARG),
    ("tree_commit", dict(max_nodes=129), _lib.ERR_ARG),
    ("tree_commit", dict(lens_out=P), _lib.ERR_ARG),
    ("tree_commit", dict(dt=3), _lib.ERR_DTYPE),
    ("tree_commit", dict(layer_stride=64), _lib.ERR_SHAPE),
    ("tree_commit", dict(page_rows=12), _lib.ERR_SHAPE),
    ("tree_commit", dict(max_len=1000), _lib.ERR_SHAPE),
    ("tree_commit", dict(k=P + 8), _lib.ERR_ALIGN),
    ("tree_commit", dict(KV=1, D=6), _lib.ERR_ALIGN),
    ("tree_commit", dict(B=65536), _lib.ERR_UNSUPPORTED),
]


@pytest.mark.parametrize("name,kw,code", BAD, ids=[f"{n}-{'-'.join(k)}" for n, k, _ in BAD])
def test_refusals(lib, name, kw, code):
    assert call(lib, name, **kw) == code
    assert _lib.last_error()


def test_workspace_sizes(lib):
    # two parts per SM of the item's rows: (o, m, l) in f32
    assert lib.b2a_tree_decode_workspace_bytes(8, 32, 8, 128, F16, 4096) >= 2 * 32 * 130 * 4
    assert lib.b2a_tree_decode_workspace_bytes(8, 32, 8, 128, F16, 64) == 0
    assert lib.b2a_tree_decode_workspace_bytes(0, 32, 8, 128, F16, 4096) == 0
    assert lib.b2a_constrain_logits_workspace_bytes(10, 128256) >= 10 * 8
    assert lib.b2a_constrain_logits_workspace_bytes(0, 5) == 0
