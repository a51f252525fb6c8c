"""GPU tests of the paged KV cache's page operators and row store against the map
kept by hand (tests/pages_util.py) and numpy: everything here moves or counts whole
numbers and bytes, so every comparison is exact; one-byte rows are quantized to the
same codes as the decode step's (the oracle's rule restated in numpy)."""
import ctypes

import numpy as np
import pytest

import cuqwen_amd as cq
from tests.conftest import tiny_config
from tests.gpu_util import Pool
from tests.pages_util import Book, DeviceMap, DevicePool, Hip, ceil, values

pytestmark = pytest.mark.gpu
L = cq.lib
KVS = [cq.KV_FP16, cq.KV_INT8, cq.KV_FP8]


@pytest.fixture
def g():
    p = Pool()
    yield p
    p.close()


def _fork(g, m, parents, children, stream=None):
    st = g.empty(4 * len(parents))
    cq.check(L.cq_pages_fork(m.arg(), g.i32(parents), g.i32(children), len(parents), st.ptr, stream))
    return st


def _trim(g, m, seqs, keep=None, stream=None):
    st = g.empty(4 * len(seqs))
    cq.check(L.cq_pages_trim(m.arg(), g.i32(seqs), None if keep is None else g.i32(keep), len(seqs), st.ptr, stream))
    return st


def _append(g, p, m, add, n_slots, stream=None):
    slots, st = g.empty(4 * max(n_slots, 1)), g.empty(16)
    cq.check(L.cq_pages_append(p.arg(), m.arg(), g.i32(add), slots.ptr if n_slots else None, n_slots, st.ptr, m.work.ptr, stream))
    return slots, st


def _compact(g, p, m, stream=None):
    remap, st = g.empty(4 * m.book.n_pages), g.empty(16)
    cq.check(L.cq_pages_compact(p.arg(), m.arg(), remap.ptr, st.ptr, m.work.ptr, stream))
    return remap, st


def _ints(b):
    return b.to_array(np.int32).tolist()


def _append_and_compare(g, p, m, add, n_slots):
    slots, st = _append(g, p, m, add, n_slots)
    want, status, moves = m.book.append(add, n_slots)
    assert _ints(st) == status
    assert n_slots == 0 or _ints(slots) == want
    m.same()
    p.move(moves)
    return status[0]


def _make(g, seed, kv=cq.KV_FP16, layers=1, n_pages=40, page=32, n_kv=1, hd=64, n_seqs=8, max_pages=12, form="own"):
    rng = np.random.default_rng(seed)
    p = DevicePool(g, rng, kv, layers, n_pages, page, n_kv, hd, form)
    return rng, p, DeviceMap(g, Book(n_pages, n_seqs, max_pages, page))


@pytest.mark.parametrize("page,n_pages,n_seqs,kv", [(32, 40, 8, 0), (64, 17, 5, 1), (128, 1, 1, 2), (32, 300, 60, 0)])
def test_a_life_of_sequences(g, page, n_pages, n_seqs, kv):
    """Random forks, appends, trims and compactions, some of them refused, each step against the model."""
    rng, p, m = _make(g, page + n_seqs, kv, 2, n_pages, page, 2, 64, n_seqs, 6)
    for step in range(25):
        what = rng.integers(0, 5)
        if what == 0:
            n = int(rng.integers(1, n_seqs + 3))
            a, b = (rng.integers(-1, n_seqs + 1, n).tolist() for _ in range(2))
            st = _fork(g, m, a, b)
            assert _ints(st) == m.book.fork(a, b)
        elif what == 1:
            n = int(rng.integers(1, n_seqs + 2))
            a = rng.integers(-1, n_seqs + 1, n).tolist()
            keep = None if rng.random() < 0.4 else rng.integers(-1, 4 * page, n).tolist()
            st = _trim(g, m, a, keep)
            assert _ints(st) == m.book.trim(a, keep)
        elif what == 2:
            remap, st = _compact(g, p, m)
            want, status, moves = m.book.compact()
            assert _ints(remap) == want and _ints(st) == status
            p.move(moves)
        else:
            add = (rng.integers(0, 2 * page, n_seqs) * (rng.random(n_seqs) < 0.6)).tolist()
            _append_and_compare(g, p, m, add, sum(add) + int(rng.integers(-1, 3)) if sum(add) else 2)
        m.same()
    p.same()


def test_append_refusals_change_nothing(g):
    rng, p, m = _make(g, 3, n_pages=10, n_seqs=6, max_pages=4)
    assert _append_and_compare(g, p, m, [33, 64, 0, 1, 0, 0], 98) == 0
    for add, n in (([0, 0, 200, 0, 0, 0], 200), ([96, 64, 0, 0, 0, 0], 159), ([0, -1, 0, 0, 0, 0], 4), ([2 ** 31 - 1] * 6, 7),
                   ([1, 1, 1, 1, 1, 1], 5), ([2 ** 30] * 6, 2 ** 20)):
        assert _append_and_compare(g, p, m, add, n) == 6
    assert _append_and_compare(g, p, m, [90, 60, 96, 1, 0, 0], 300) == 5   # too few pages
    m.book.table[0][1] = 10                                                # a last page outside the pool
    m.upload()
    assert _append_and_compare(g, p, m, [1, 0, 0, 0, 0, 0], 4) == 6
    m.book.table[0][1] = -7
    m.upload()
    assert _append_and_compare(g, p, m, [1, 0, 0, 0, 0, 0], 4) == 6
    assert _append_and_compare(g, p, m, [0, 1, 0, 0, 0, 0], 4) == 0        # the others go on
    m.book.len[3] = -5
    m.upload()
    assert _append_and_compare(g, p, m, [0, 0, 1, 0, 0, 0], 4) == 6
    m.book.len[3] = 4 * 32 + 1
    m.upload()
    assert _append_and_compare(g, p, m, [0, 0, 1, 0, 0, 0], 4) == 6
    for st in (_fork(g, m, [3], [4]), _trim(g, m, [3])):
        assert _ints(st) == [6]
    assert m.book.fork([3], [4]) == [6] and m.book.trim([3]) == [6]
    m.same()
    assert _append_and_compare(g, p, m, [0] * 6, 0) == 6
    p.same()


def test_bad_table_entries_are_passed_over(g):
    """Ids outside the pool in the middle of a row: nothing is counted or moved for them."""
    rng, p, m = _make(g, 4, n_pages=9, n_seqs=4, max_pages=4)
    assert _append_and_compare(g, p, m, [128, 30, 0, 0], 158) == 0
    m.book.table[0][1], m.book.table[0][2] = -3, 9
    m.upload()
    assert _ints(_fork(g, m, [0], [2])) == m.book.fork([0], [2])
    m.same()
    assert _ints(_trim(g, m, [0, 1])) == m.book.trim([0, 1])
    m.same()
    remap, st = _compact(g, p, m)
    want, status, moves = m.book.compact()
    assert _ints(remap) == want and _ints(st) == status
    p.move(moves)
    m.same()
    p.same()


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("form", ["own", "cache", "wide"])
@pytest.mark.parametrize("page,hd,n_kv,tokens", [(32, 64, 2, 5), (64, 128, 3, 33), (128, 64, 1, 96), (64, 128, 1, 64)])
def test_copy_on_write_bytes(g, kv, form, page, hd, n_kv, tokens):
    """Forks of a sequence of `tokens` tokens: whole tiles are copied, the rest of a page is left."""
    rng, p, m = _make(g, 5, kv, 3, 9, page, n_kv, hd, 6, 3, form)
    _append_and_compare(g, p, m, [tokens, 0, 0, 0, 0, 0], tokens)
    assert _ints(_fork(g, m, [0, 0, 0], [1, 3, 5])) == m.book.fork([0, 0, 0], [1, 3, 5])
    assert _append_and_compare(g, p, m, [1, 2, 0, 0, 0, 1], 4) == 0
    p.same()


@pytest.mark.parametrize("n_pages,n_seqs", [(4096, 1024), (9001, 3), (65536, 700)])
def test_large_maps(g, n_pages, n_seqs):
    """More pages than one pass of the planning block, as many sequences as it has threads."""
    rng, p, m = _make(g, 6, cq.KV_INT8, 1, n_pages, 32, 1, 64, n_seqs, n_pages // n_seqs)
    most = (n_pages // n_seqs) * 32
    assert _append_and_compare(g, p, m, rng.integers(most // 2, most + 1, n_seqs).tolist(), n_seqs * most) == 0
    gone = rng.permutation(n_seqs)[:ceil(n_seqs, 2)].tolist()
    assert _ints(_trim(g, m, gone)) == m.book.trim(gone)
    remap, st = _compact(g, p, m)
    want, status, moves = m.book.compact()
    assert _ints(remap) == want and _ints(st) == status and status[2] > 0
    p.move(moves)
    m.same()
    keep = [s for s in range(n_seqs) if s not in gone]
    pairs = [(keep[i % len(keep)], c) for i, c in enumerate(gone)] if keep else []
    if pairs:
        a, b = [x for x, _ in pairs], [y for _, y in pairs]
        assert _ints(_fork(g, m, a, b)) == m.book.fork(a, b)
        _append_and_compare(g, p, m, [1 if n < most else 0 for n in m.book.len], n_seqs)
    m.same()
    p.same()


@pytest.mark.parametrize("kv", KVS)
def test_copy_between_pools(g, kv):
    rng = np.random.default_rng(7)
    a = DevicePool(g, rng, kv, 2, 7, 64, 2, 128, "cache")
    b = DevicePool(g, rng, kv, 2, 5, 64, 2, 128, "own")
    src, dst = [6, 0, -1, 3, 2, 7, 0, 1], [4, 1, 2, 5, 3, 0, 2, 3]
    #          ok  ok  E  E  dup  E  dup dup: 2 is named by a pair that is itself refused
    st = g.empty(4 * len(src))
    cq.check(L.cq_pages_copy(a.arg(), b.arg(), g.i32(src), g.i32(dst), len(src), st.ptr, None))
    assert _ints(st) == [0, 0, 6, 6, 1, 6, 1, 1]
    for s, d in ((6, 4), (0, 1)):
        b._move(s, d, 64, a)
    b.same()
    a.same()


def test_copy_within_a_pool(g):
    rng = np.random.default_rng(8)
    a = DevicePool(g, rng, cq.KV_FP16, 3, 12, 32, 2, 64, "wide")
    src, dst = [0, 1, 2, 5, 5, 7, 4], [3, 2, 6, 8, 9, 7, 4]
    #          ok  2 is a source  ok  ok ok itself itself
    st = g.empty(4 * len(src))
    cq.check(L.cq_pages_copy(a.arg(), a.arg(), g.i32(src), g.i32(dst), len(src), st.ptr, None))
    assert _ints(st) == [0, 1, 0, 0, 0, 0, 0]
    a.move([(0, 3), (2, 6), (5, 8), (5, 9)])
    a.same()


def test_copy_of_many_pages(g):
    rng = np.random.default_rng(9)
    a = DevicePool(g, rng, cq.KV_FP8, 1, 4200, 32, 1, 64)
    b = DevicePool(g, rng, cq.KV_FP8, 1, 4200, 32, 1, 64, "wide")
    src, dst = rng.integers(0, 4200, 4096).tolist(), rng.permutation(4200)[:4096].tolist()
    st = g.empty(4 * 4096)
    cq.check(L.cq_pages_copy(a.arg(), b.arg(), g.i32(src), g.i32(dst), 4096, st.ptr, None))
    assert not any(_ints(st))
    for s, d in zip(src, dst):
        b._move(s, d, 32, a)
    b.same()


def _codes(x, kv):
    """Codes and scales of rows [..., hd] (fp16), in 32 bits as the library forms them."""
    f = x.astype(np.float32)
    s = np.abs(f).max(-1) / np.float32(127 if kv == cq.KV_INT8 else 448)
    v = f / np.where(s > 0, s, np.float32(1))[..., None]
    if kv == cq.KV_INT8:
        return np.clip(np.rint(v), -127, 127).astype(np.int8), s
    table = values(np.arange(127, dtype=np.uint8).view(np.int8), kv)   # 0 .. 448, ascending
    a = np.abs(v).astype(np.float64)
    hi = np.searchsorted(table, a).clip(1, 126)
    lo = hi - 1
    pick = np.where(a - table[lo] < table[hi] - a, lo, hi)
    pick = np.where(a - table[lo] == table[hi] - a, np.where(lo % 2 == 0, lo, hi), pick).astype(np.uint8)
    return (pick | (np.signbit(v).astype(np.uint8) << 7)).view(np.int8), s


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("form,page,hd,n_kv", [("own", 32, 64, 2), ("wide", 64, 128, 3), ("cache", 128, 128, 1)])
@pytest.mark.parametrize("tokens", [1, 31, 64, 100])
def test_store_and_load_rows(g, kv, form, page, hd, n_kv, tokens):
    rng = np.random.default_rng(tokens + hd)
    p = DevicePool(g, rng, kv, 2, 9, page, n_kv, hd, form)
    total = p.n_pages * page
    # consecutive from a tile's beginning, scattered, or with slots outside the pool among them
    for slots in (list(range(32, 32 + tokens)), rng.permutation(total)[:tokens].tolist(), None):
        if slots is None:
            slots = rng.permutation(total)[:tokens].tolist()
            for i, bad in zip(range(0, tokens, 7), [-1, total, 2 ** 31 - 1, -2 ** 31] * 9):
                slots[i] = bad
        stride = n_kv * hd + 8 * int(rng.integers(0, 3))
        rows = [(rng.standard_normal((tokens, stride)) * np.exp(rng.standard_normal((tokens, 1)))).astype(np.float16) for _ in range(2)]
        for r in rows:
            r[0, :hd] = 0          # a zero row
        layer = int(rng.integers(0, 2))
        cq.check(L.cq_paged_kv_store(p.arg(), layer, g.put(rows[0]), g.put(rows[1]), stride, g.i32(slots), tokens, None))
        back = [g.put(np.full((tokens, stride), -7, np.float16)) for _ in range(2)]
        cq.check(L.cq_paged_kv_load(p.arg(), layer, back[0], back[1], stride, g.i32(slots), tokens, None))
        for k in range(2):
            x = rows[k][:, :n_kv * hd].reshape(tokens, n_kv, hd)
            code, s = (x, None) if kv == cq.KV_FP16 else _codes(x, kv)
            for t, slot in enumerate(slots):
                if not 0 <= slot < total:
                    continue
                at = p.at[layer, slot // page]
                p.host[k][at[:, None] + p.offsets(k)[slot % page]] = code[t]
                if s is not None:
                    p.scales[k][at // hd + slot % page] = s[t]
            want = np.full((tokens, stride), -7, np.float16)
            v = x if s is None else (values(code, kv).astype(np.float32) * s[..., None]).astype(np.float16)
            ok = [t for t, slot in enumerate(slots) if 0 <= slot < total]
            want[ok, :n_kv * hd] = v.reshape(tokens, -1)[ok]
            got = np.zeros_like(want)
            cq.check(L.cq_memcpy_d2h(got.ctypes.data, back[k], got.nbytes))
            assert np.array_equal(got, want)
        p.same()


def test_a_states_cache_as_pages(g):
    """Positions of a state's own cache read as pages, and the prompt copied into a pool."""
    for kv in KVS:
        cfg = tiny_config(max_seq_len=544)
        w = cq.synth_weights(cfg, 5)
        st = cq.State(cfg, w, kv_dtype=kv)
        st.prefill(list(range(1, 101)))
        for page in (32, 64, 512):
            v = st.kv_pages(page)
            assert (v.n_pages, v.page_tokens, v.n_layers, v.kv_dtype) == (544 // page, page, cfg.n_layers, kv)
            slots, hd, n_kv = g.i32(list(range(100))), cfg.head_dim, cfg.n_kv_heads
            k, x = g.empty(100 * n_kv * hd * 2), g.empty(100 * n_kv * hd * 2)
            for layer in range(cfg.n_layers):
                cq.check(L.cq_paged_kv_load(ctypes.byref(v), layer, k.ptr, x.ptr, n_kv * hd, slots, 100, None))
                for h in range(n_kv):
                    for kind, b in ((0, k), (1, x)):
                        got = b.to_array(np.uint16, (100, n_kv, hd))[:, h]
                        assert np.array_equal(got, st.kv_read(layer, h, kind, 100).view(np.uint16))
        v = st.kv_pages(32)
        p = DevicePool(g, np.random.default_rng(1), kv, cfg.n_layers, 6, 32, cfg.n_kv_heads, cfg.head_dim)
        status = g.empty(16)
        cq.check(L.cq_pages_copy(ctypes.byref(v), p.arg(), g.i32([0, 1, 2, 3]), g.i32([5, 0, 3, 2]), 4, status.ptr, None))
        assert not any(_ints(status))
        order = np.array([5, 0, 3, 2])[np.arange(100) // 32] * 32 + np.arange(100) % 32
        k, x = g.empty(100 * n_kv * hd * 2), g.empty(100 * n_kv * hd * 2)
        cq.check(L.cq_paged_kv_load(p.arg(), 1, k.ptr, x.ptr, n_kv * hd, g.i32(order), 100, None))
        for h in range(n_kv):
            assert np.array_equal(x.to_array(np.uint16, (100, n_kv, hd))[:, h], st.kv_read(1, h, 1, 100).view(np.uint16))
        for bad in (0, 16, 48, 1024):
            with pytest.raises(cq.CuQwenError, match="EINVAL"):
                st.kv_pages(bad)
        st.free()
        w.free()


def test_captured_page_operators(g):
    """One graph of fork, append, trim and compact, replayed with other work between, each replay against the model."""
    rng, p, m = _make(g, 11, cq.KV_INT8, 2, 60, 32, 2, 64, 10, 6)
    hip = Hip()
    stream = hip.stream()
    assert _append_and_compare(g, p, m, [70] + [0] * 9, 70) == 0
    slots, st, remap = g.empty(4 * 8), g.empty(4 * (4 + 4 + 4 + 4)), g.empty(4 * 60)
    parents, children, add = g.i32([0, 0, 0, 0]), g.i32([2, 3, 4, 5]), g.i32([0, 1] + [2] * 4 + [0] * 4)
    drop = g.i32([2, 4, 3, 5])
    cq.synchronize()

    def body():
        cq.check(L.cq_pages_fork(m.arg(), parents, children, 4, st.value, stream))
        cq.check(L.cq_pages_append(p.arg(), m.arg(), add, slots.ptr, 8, st.value + 16, m.work.ptr, stream))
        cq.check(L.cq_pages_trim(m.arg(), drop, None, 4, st.value + 32, stream))
        cq.check(L.cq_pages_compact(p.arg(), m.arg(), remap.ptr, st.value + 48, m.work.ptr, stream))

    graph = hip.capture(stream, body)
    for replay in range(4):
        hip.launch(graph, stream)
        hip.wait(stream)
        a = m.book.fork([0] * 4, [2, 3, 4, 5])
        want, b, moves = m.book.append([0, 1] + [2] * 4 + [0] * 4, 8)
        p.move(moves)
        c = m.book.trim([2, 4, 3, 5])
        after, d, moves = m.book.compact()
        p.move(moves)
        assert _ints(st) == a + b + c + d and _ints(slots) == want and _ints(remap) == after
        m.same()
        p.same()
        _append_and_compare(g, p, m, [replay, 0] + [0] * 8, 8)   # work of the caller's own between the replays
    hip.drop(stream, [graph])


def test_two_maps_on_two_streams(g):
    """Two pools, maps and workspaces at once."""
    hip = Hip()
    streams = [hip.stream(), hip.stream()]
    sets = [_make(g, 20 + i, cq.KV_FP16, 2, 30, 64, 1, 64, 6, 5) for i in range(2)]
    cq.synchronize()
    got = []
    for step in range(6):
        for (rng, p, m), s in zip(sets, streams):
            add = rng.integers(0, 40, 6).tolist()
            got.append((p, m, add, _append(g, p, m, add, 240, s)))
    for s in streams:
        hip.wait(s)
    for p, m, add, (slots, st) in got:
        want, status, moves = m.book.append(add, 240)
        p.move(moves)
        assert _ints(st) == status and _ints(slots) == want
    for rng, p, m in sets:
        m.same()
        p.same()
    for s in streams:
        hip.drop(s)
