"""Host-side refusals of normed heads, the 4-bit cache and sampled verification: every
case returns before any CUDA call (the addresses are never read)."""
import pytest

from alpacca_open_sourced_by_jt_b200 import _lib, build

P = 1 << 20
F16, BF16, F32 = _lib.F16, _lib.BF16, _lib.F32


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


CALLS = {
    "norm_rope_append_paged": dict(q=P, qs=512, k=P, ks=128, v=P, vs=128, dt=F32, bq=None, bk=None, bv=None, wq=P,
                                   wk=P, eps=1e-6, cos=P, sin=P, tab_rows=16, pos=P, slot=P, kp=P, vp=P, n_pages=4,
                                   page_rows=16, page_stride=0, kv_dt=F16, q_out=P, n_tok=0, H=8, KV=2, D=64, n_rot=64,
                                   style=0, stream=None),
    "rope_append_q4": dict(q=P, qs=512, k=P, ks=128, v=P, vs=128, dt=F32, bq=None, bk=None, bv=None, wq=P, wk=P,
                           eps=1e-6, cos=P, sin=P, tab_rows=16, pos=P, slot=P, pool=P, n_pages=4, page_rows=16,
                           page_bytes=0, q_out=P, qo_dt=F16, n_tok=0, H=8, KV=2, D=64, n_rot=64, style=0, stream=None),
    "q4_rows": dict(pool=P, n_pages=4, page_rows=16, page_bytes=0, slot=P, k=P, v=P, dt=F16, n_tok=0, KV=2, D=64,
                    stream=None),
    "tree_decode_q4": dict(q=P, qs=0, pool=P, n_pages=64, page_rows=16, page_bytes=0, table=P, stride=8, width=8,
                           lens=P, cu=P, parents=P, out=P, lse=None, ws=P, ws_bytes=1 << 30, B=2, n_tok=0, max_nodes=8,
                           H=8, KV=2, D=64, dt=F16, scale=0.125, max_len=128, stream=None),
    "tree_commit_q4": dict(picks=P, tokens=P, parents=None, cu=P, lens=P, table=P, stride=8, width=8, pool=P, L=2,
                           layer_bytes=1 << 20, n_pages=64, page_rows=16, page_bytes=0, KV=2, D=64, B=2, n_tok=8,
                           max_nodes=8, max_len=128, path=P, acc=P, next=P, lens_out=2 * P, stream=None),
    "verify_picks": dict(x=P, xs=1000, dt=F32, draft=P, ds=1000, cu=P, parents=None, tokens=P, u=P, d=P, T=None,
                         picks=P, B=2, n_rows=0, max_nodes=4, V=1000, stream=None),
}


def call(lib, name, **kw):
    args = dict(CALLS[name])
    assert set(kw) <= set(args)
    args.update(kw)
    return getattr(lib, "b2a_" + name)(*args.values())


@pytest.mark.parametrize("name", ["norm_rope_append_paged", "rope_append_q4", "q4_rows", "tree_decode_q4",
                                  "verify_picks"])
def test_no_tokens_is_a_successful_no_op(lib, name):
    assert call(lib, name) == _lib.OK


APPEND = [
    (dict(q=None), _lib.ERR_ARG), (dict(q_out=None), _lib.ERR_ARG), (dict(cos=None), _lib.ERR_ARG),
    (dict(slot=None), _lib.ERR_ARG), (dict(n_tok=-1), _lib.ERR_ARG), (dict(KV=0), _lib.ERR_ARG),
    (dict(tab_rows=0), _lib.ERR_ARG), (dict(n_pages=0), _lib.ERR_ARG), (dict(D=96), _lib.ERR_UNSUPPORTED),
    (dict(D=63), _lib.ERR_UNSUPPORTED), (dict(style=2), _lib.ERR_ARG), (dict(n_rot=66), _lib.ERR_SHAPE),
    (dict(n_rot=80), _lib.ERR_SHAPE), (dict(n_rot=-16), _lib.ERR_SHAPE), (dict(n_rot=24), _lib.ERR_SHAPE),
    (dict(dt=9), _lib.ERR_DTYPE), (dict(page_rows=24), _lib.ERR_SHAPE), (dict(page_rows=0), _lib.ERR_SHAPE),
    (dict(eps=-1e-6), _lib.ERR_ARG), (dict(eps=float("nan")), _lib.ERR_ARG), (dict(eps=float("inf")), _lib.ERR_ARG),
    (dict(qs=511), _lib.ERR_SHAPE), (dict(ks=64), _lib.ERR_SHAPE), (dict(qs=513), _lib.ERR_ALIGN),
    (dict(vs=130), _lib.ERR_ALIGN), (dict(dt=F16, vs=132), _lib.ERR_ALIGN), (dict(k=P + 4), _lib.ERR_ALIGN),
    (dict(wq=P + 4), _lib.ERR_ALIGN), (dict(bk=P + 8), _lib.ERR_ALIGN), (dict(sin=P + 4), _lib.ERR_ALIGN),
    (dict(q_out=P + 8), _lib.ERR_ALIGN),
]
BAD = [(name, kw, code) for name in ("norm_rope_append_paged", "rope_append_q4") for kw, code in APPEND] + [
    ("norm_rope_append_paged", dict(kv_dt=7), _lib.ERR_DTYPE),
    ("norm_rope_append_paged", dict(page_stride=100), _lib.ERR_SHAPE),
    ("norm_rope_append_paged", dict(page_stride=16 * 128 + 4), _lib.ERR_ALIGN),
    ("norm_rope_append_paged", dict(vp=P + 8), _lib.ERR_ALIGN),
    ("rope_append_q4", dict(pool=None), _lib.ERR_ARG),
    ("rope_append_q4", dict(qo_dt=F32), _lib.ERR_DTYPE),
    ("rope_append_q4", dict(style=1, n_rot=32), _lib.ERR_SHAPE),
    ("rope_append_q4", dict(page_bytes=2 * 18 * 64 - 16), _lib.ERR_SHAPE),
    ("rope_append_q4", dict(page_bytes=2 * 18 * 64 + 8), _lib.ERR_ALIGN),
    ("rope_append_q4", dict(page_rows=8), _lib.ERR_SHAPE),
    ("q4_rows", dict(pool=None), _lib.ERR_ARG),
    ("q4_rows", dict(v=None), _lib.ERR_ARG),
    ("q4_rows", dict(n_tok=-1), _lib.ERR_ARG),
    ("q4_rows", dict(D=32), _lib.ERR_UNSUPPORTED),
    ("q4_rows", dict(dt=8), _lib.ERR_DTYPE),
    ("q4_rows", dict(page_rows=40), _lib.ERR_SHAPE),
    ("q4_rows", dict(k=P + 2), _lib.ERR_ALIGN),
    ("tree_decode_q4", dict(q=None), _lib.ERR_ARG),
    ("tree_decode_q4", dict(pool=None), _lib.ERR_ARG),
    ("tree_decode_q4", dict(cu=None), _lib.ERR_ARG),
    ("tree_decode_q4", dict(B=0), _lib.ERR_ARG),
    ("tree_decode_q4", dict(n_tok=-1), _lib.ERR_ARG),
    ("tree_decode_q4", dict(max_nodes=0), _lib.ERR_ARG),
    ("tree_decode_q4", dict(max_nodes=129), _lib.ERR_ARG),
    ("tree_decode_q4", dict(max_len=0), _lib.ERR_ARG),
    ("tree_decode_q4", dict(H=9), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(D=96), _lib.ERR_UNSUPPORTED),
    ("tree_decode_q4", dict(dt=F32), _lib.ERR_DTYPE),
    ("tree_decode_q4", dict(dt=5), _lib.ERR_DTYPE),
    ("tree_decode_q4", dict(scale=0.0), _lib.ERR_ARG),
    ("tree_decode_q4", dict(scale=float("inf")), _lib.ERR_ARG),
    ("tree_decode_q4", dict(page_rows=8), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(page_rows=48), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(max_len=129), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(stride=4), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(table=None, n_pages=1, page_rows=512), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(table=None, page_rows=112), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(table=None, page_rows=136), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(page_bytes=64), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(page_bytes=(1 << 20) + 4), _lib.ERR_ALIGN),
    ("tree_decode_q4", dict(page_rows=1 << 30), _lib.ERR_UNSUPPORTED),
    ("tree_decode_q4", dict(qs=100), _lib.ERR_SHAPE),
    ("tree_decode_q4", dict(qs=516), _lib.ERR_ALIGN),
    ("tree_decode_q4", dict(q=P + 2), _lib.ERR_ALIGN),
    ("tree_decode_q4", dict(ws=P + 4), _lib.ERR_ALIGN),
    ("tree_decode_q4", dict(H=400, KV=2, n_tok=1), _lib.ERR_UNSUPPORTED),
    ("tree_decode_q4", dict(n_tok=4, ws_bytes=64, max_len=4096, width=256, stride=256), _lib.ERR_WORKSPACE),
    ("tree_decode_q4", dict(n_tok=4, ws=None, max_len=4096, width=256, stride=256), _lib.ERR_WORKSPACE),
    ("tree_commit_q4", dict(path=None), _lib.ERR_ARG),
    ("tree_commit_q4", dict(pool=None), _lib.ERR_ARG),
    ("tree_commit_q4", dict(L=0), _lib.ERR_ARG),
    ("tree_commit_q4", dict(max_nodes=129), _lib.ERR_ARG),
    ("tree_commit_q4", dict(lens_out=P), _lib.ERR_ARG),
    ("tree_commit_q4", dict(layer_bytes=64), _lib.ERR_SHAPE),
    ("tree_commit_q4", dict(layer_bytes=(1 << 20) + 8), _lib.ERR_SHAPE),
    ("tree_commit_q4", dict(page_rows=24), _lib.ERR_SHAPE),
    ("tree_commit_q4", dict(max_len=1000), _lib.ERR_SHAPE),
    ("tree_commit_q4", dict(pool=P + 8), _lib.ERR_ALIGN),
    ("tree_commit_q4", dict(D=80), _lib.ERR_UNSUPPORTED),
    ("tree_commit_q4", dict(B=65536), _lib.ERR_UNSUPPORTED),
    ("verify_picks", dict(x=None), _lib.ERR_ARG),
    ("verify_picks", dict(u=None), _lib.ERR_ARG),
    ("verify_picks", dict(d=None), _lib.ERR_ARG),
    ("verify_picks", dict(picks=None), _lib.ERR_ARG),
    ("verify_picks", dict(V=0), _lib.ERR_ARG),
    ("verify_picks", dict(B=0), _lib.ERR_ARG),
    ("verify_picks", dict(n_rows=-1), _lib.ERR_ARG),
    ("verify_picks", dict(max_nodes=0), _lib.ERR_ARG),
    ("verify_picks", dict(max_nodes=129), _lib.ERR_ARG),
    ("verify_picks", dict(dt=4), _lib.ERR_DTYPE),
    ("verify_picks", dict(xs=999), _lib.ERR_SHAPE),
    ("verify_picks", dict(ds=999), _lib.ERR_SHAPE),
    ("verify_picks", dict(V=2000001, xs=1 << 22, ds=1 << 22), _lib.ERR_UNSUPPORTED),
    ("verify_picks", dict(B=1 << 30), _lib.ERR_UNSUPPORTED),
    ("verify_picks", dict(x=P + 2), _lib.ERR_ALIGN),
    ("verify_picks", dict(draft=P + 2), _lib.ERR_ALIGN),
]


@pytest.mark.parametrize("name,kw,code", BAD, ids=[f"{n}-{'-'.join(k)}-{i}" for i, (n, k, _) in enumerate(BAD)])
def test_refusals(lib, name, kw, code):
    assert call(lib, name, **kw) == code
    assert _lib.last_error()


def test_workspace_sizes(lib):
    size = lib.b2a_tree_decode_q4_workspace_bytes
    assert size(8, 32, 8, 128, 4096) >= 2 * 32 * 130 * 4  # two parts per SM of the item's rows: (o, m, l) in f32
    assert size(8, 32, 8, 128, 64) == 0
    assert size(0, 32, 8, 128, 4096) == 0 and size(8, 30, 8, 128, 4096) == 0
