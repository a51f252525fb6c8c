"""CPU tests of the paged KV cache's host side: layouts, workspace sizes and the
refusals that need no device (every call here is refused, or has nothing to do,
before it touches the GPU)."""
import ctypes

import pytest

import cuqwen_amd as cq
from tests.pages_util import Book, ceil

A = 1 << 20   # stands for an aligned device address; never read


def _pool(kv=0, layers=2, pages=8, page=64, n_kv=2, hd=64, **kw):
    p = cq.kv_pages(page, n_kv, hd, pages, layers, kv, A, 2 * A, 3 * A, 4 * A)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _map(pages=8, seqs=4, width=4, page=64, **kw):
    m = cq.page_map(A, 2 * A, 3 * A, pages, seqs, width, page)
    for k, v in kw.items():
        setattr(m, k, v)
    return m


def B(x):
    return ctypes.byref(x) if x is not None else None


def refused(rc, code="EINVAL"):
    with pytest.raises(cq.CuQwenError, match=code):
        cq.check(rc)


@pytest.mark.parametrize("kv,es", [(0, 2), (1, 1), (2, 1)])
def test_layout(kv, es):
    p = cq.kv_pages(32, 8, 128, 5, 3, kv)
    assert (p.head_stride, p.page_stride, p.layer_stride) == (32 * 128, 8 * 32 * 128, 5 * 8 * 32 * 128)
    assert cq.kv_pages_bytes(p) == (3 * 5 * 8 * 32 * 128 * es, 0 if kv == 0 else 3 * 5 * 8 * 32 * 4)
    assert (p.kv_dtype, p.n_layers, p.n_pages, p.page_tokens, p.n_kv_heads, p.head_dim) == (kv, 3, 5, 32, 8, 128)


@pytest.mark.parametrize("bad", [dict(kv=3), dict(kv=-1), dict(layers=0), dict(pages=0), dict(pages=(1 << 20) + 1), dict(page=16),
                                 dict(page=48), dict(page=65536), dict(n_kv=0), dict(n_kv=65), dict(hd=96), dict(hd=0),
                                 dict(pages=1 << 16, page=32768)])
def test_layout_refusals(bad):
    a = dict(kv=0, layers=2, pages=8, page=64, n_kv=2, hd=64)
    a.update(bad)
    with pytest.raises(cq.CuQwenError, match="EINVAL"):
        cq.kv_pages(a["page"], a["n_kv"], a["hd"], a["pages"], a["layers"], a["kv"])


BAD_POOLS = [dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 2), dict(kv_dtype=1, k_scale=None), dict(kv_dtype=2, v_scale=None),
             dict(kv_dtype=1, k_scale=A + 4), dict(page_stride=64 * 64), dict(head_stride=32 * 64), dict(layer_stride=64 * 64),
             dict(page_stride=2 * 64 * 64 + 8), dict(head_stride=-64 * 64), dict(page_stride=1 << 60), dict(n_pages=0),
             dict(page_tokens=33), dict(head_dim=32), dict(n_kv_heads=0), dict(n_layers=0), dict(kv_dtype=7)]
BAD_MAPS = [dict(ref=None), dict(table=None), dict(len=None), dict(n_seqs=0), dict(n_seqs=1025), dict(n_pages=0), dict(max_pages=0),
            dict(max_pages=1 << 25), dict(page_tokens=31), dict(page_tokens=0)]


def _pool_calls(p):
    L, m = cq.lib, _map()
    good = _pool()
    yield L.cq_pages_append(B(p), B(m), A, A, 4, A, A, None)
    yield L.cq_pages_compact(B(p), B(m), A, A, A, None)
    yield L.cq_pages_copy(B(p), B(good), A, A, 1, A, None)
    yield L.cq_pages_copy(B(good), B(p), A, A, 1, A, None)
    yield L.cq_paged_kv_store(B(p), 0, A, A, 128, A, 1, None)
    yield L.cq_paged_kv_load(B(p), 0, A, A, 128, A, 1, None)
    yield L.cq_prefix_attention_decode(A, 256, A, 256, B(p), A, 1, A, B(good), A, 1, None, A, 1, 0, 4, A, None)
    yield L.cq_prefix_attention_decode(A, 256, A, 256, B(good), A, 1, A, B(p), A, 1, None, A, 1, 0, 4, A, None)


@pytest.mark.parametrize("bad", BAD_POOLS + [None])
def test_bad_pools_are_refused(bad):
    for rc in _pool_calls(None if bad is None else _pool(**bad)):
        refused(rc)


@pytest.mark.parametrize("bad", BAD_MAPS + [None])
def test_bad_maps_are_refused(bad):
    L, p, m = cq.lib, _pool(), None if bad is None else _map(**bad)
    refused(L.cq_pages_fork(B(m), A, A, 1, A, None))
    refused(L.cq_pages_trim(B(m), A, None, 1, A, None))
    refused(L.cq_pages_append(B(p), B(m), A, A, 4, A, A, None))
    refused(L.cq_pages_compact(B(p), B(m), A, A, A, None))


def test_pool_and_map_must_agree():
    L = cq.lib
    for m in (_map(pages=9), _map(page=32)):
        refused(L.cq_pages_append(B(_pool()), B(m), A, A, 4, A, A, None))
        refused(L.cq_pages_compact(B(_pool()), B(m), A, A, A, None))


def test_arguments_of_the_page_operators():
    L, p, m = cq.lib, _pool(), _map()
    for n in (-1, 1025):
        refused(L.cq_pages_fork(B(m), A, A, n, A, None))
        refused(L.cq_pages_trim(B(m), A, None, n, A, None))
    for a in ((None, A, A), (A, None, A), (A, A, None)):
        refused(L.cq_pages_fork(B(m), a[0], a[1], 1, a[2], None))
        refused(L.cq_pages_copy(B(p), B(p), a[0], a[1], 1, a[2], None))
    refused(L.cq_pages_trim(B(m), None, None, 1, A, None))
    refused(L.cq_pages_trim(B(m), A, None, 1, None, None))
    for a in ((None, A, 4, A, A), (A, None, 4, A, A), (A, A, -1, A, A), (A, A, 4, None, A), (A, A, 4, A, None), (A, A, 4, A, A + 4)):
        refused(L.cq_pages_append(B(p), B(m), *a, None))
    for a in ((None, A, A), (A, None, A), (A, A, None), (A, A, A + 8)):
        refused(L.cq_pages_compact(B(p), B(m), *a, None))
    for n in (-1, 4097):
        refused(L.cq_pages_copy(B(p), B(p), A, A, n, A, None))
    for other in (_pool(kv=1), _pool(layers=3), _pool(page=32), _pool(n_kv=1), _pool(hd=128)):
        refused(L.cq_pages_copy(B(p), B(other), A, A, 1, A, None))
    # nothing to do
    cq.check(L.cq_pages_fork(B(m), None, None, 0, None, None))
    cq.check(L.cq_pages_trim(B(m), None, None, 0, None, None))
    cq.check(L.cq_pages_copy(B(p), B(p), None, None, 0, None, None))


def test_arguments_of_the_row_store():
    L, p = cq.lib, _pool()
    for f in (L.cq_paged_kv_store, L.cq_paged_kv_load):
        for layer in (-1, 2):
            refused(f(B(p), layer, A, A, 128, A, 1, None))
        for a in ((None, A, 128, A, 1), (A, None, 128, A, 1), (A + 8, A, 128, A, 1), (A, A + 2, 128, A, 1), (A, A, 120, A, 1),
                  (A, A, 132, A, 1), (A, A, -128, A, 1), (A, A, 128, None, 1), (A, A, 128, A, -1), (A, A, 128, A, (1 << 24) + 1)):
            refused(f(B(p), 0, *a, None))
        cq.check(f(B(p), 0, None, None, 0, None, 0, None))


def test_arguments_of_the_attention():
    L, p = cq.lib, _pool()
    good = dict(q=A, qs=256, out=2 * A, os=256, pre=p, pt=A, pp=1, pl=A, own=p, t=A, mp=1, st=None, ln=A, batch=1, layer=0, heads=4, ws=A)

    def call(**kw):
        a = dict(good, **kw)
        return L.cq_prefix_attention_decode(a["q"], a["qs"], a["out"], a["os"], B(a["pre"]), a["pt"], a["pp"], a["pl"], B(a["own"]),
                                            a["t"], a["mp"], a["st"], a["ln"], a["batch"], a["layer"], a["heads"], a["ws"], None)

    for bad in (dict(q=None), dict(out=None), dict(pt=None), dict(pl=None), dict(t=None), dict(ln=None), dict(ws=None), dict(q=A + 8),
                dict(out=A + 4), dict(ws=A + 8), dict(qs=248), dict(qs=260), dict(os=128), dict(os=-256), dict(pp=0), dict(mp=0),
                dict(pp=-1), dict(batch=-1), dict(batch=1025), dict(layer=-1), dict(layer=2), dict(heads=0), dict(heads=3),
                dict(heads=34), dict(own=_pool(kv=1)), dict(own=_pool(n_kv=1)), dict(own=_pool(hd=128)), dict(pre=_pool(layers=1), layer=1)):
        refused(call(**bad))
    # a table's row of more than 2^30 positions (the pool's pages have 64)
    for bad in (dict(pp=(1 << 24) + 1), dict(mp=(1 << 24) + 1), dict(pp=(1 << 31) - 1), dict(mp=(1 << 31) - 1)):
        refused(call(**bad))
    cq.check(call(batch=0, q=None, out=None))


def test_workspace_sizes():
    L = cq.lib
    assert L.cq_pages_workspace_bytes(B(_map())) > 0 and L.cq_pages_workspace_bytes(None) == 0
    f = L.cq_prefix_attention_workspace_bytes
    assert 0 < f(1, 4, 2, 64) <= f(2, 4, 2, 64) <= f(64, 28, 4, 128) <= f(1024, 28, 4, 128)
    assert f(0, 4, 2, 64) >= 0
    for bad in ((-1, 4, 2, 64), (1025, 4, 2, 64), (1, 4, 3, 64), (1, 40, 2, 64), (1, 4, 2, 96), (1, 0, 2, 64), (1, 4, 0, 64)):
        assert f(*bad) == 0


def test_the_model_of_the_map():
    """The hand-kept map that the GPU tests compare with, on a case worked out on paper."""
    b = Book(8, 4, 4, 32)
    assert b.append([40, 0, 0, 0], 40)[1] == [0, 2, 0, 40] and b.table[0][:2] == [0, 1]
    assert b.fork([0, 0, 1], [1, 2, 2]) == [0, 0, 1]          # the last: its parent is a child, its child named before
    assert b.ref[:2] == [3, 3]
    slots, st, moves = b.append([1, 1, 1, 0], 4)              # three writers to page 1: the last keeps it
    assert st == [0, 2, 2, 3] and moves == [(1, 2, 32), (1, 3, 32)] and slots == [72, 104, 40, -1] and b.ref[:4] == [3, 1, 1, 1]
    assert b.trim([0, 2, 0], [32, 0, 1]) == [0, 0, 1] and b.ref[:4] == [2, 0, 0, 1] and b.len == [32, 41, 0, 0]
    remap, st, moves = b.compact()
    assert st == [0, 2, 1, 0] and moves == [(3, 1)] and b.table[1][:2] == [0, 1] and remap[:4] == [0, -1, -1, 1]
    assert b.append([200, 0, 0, 0], 999)[1][0] == 6 and ceil(65, 32) == 3
