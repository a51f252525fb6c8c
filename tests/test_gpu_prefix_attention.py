"""GPU tests of the batch attention over a shared prefix (cq_prefix_attention_decode)
against the formula in 64 bits.

Tolerance, per output element, with w the softmax weights and A = sum w |v|:
  the output's rounding to fp16        2^-11 |out| + 2^-25
  each weight's rounding to fp16       2^-11 A, and 2^-25 |v| for each key whose
                                       exponential lies in fp16's subnormals (times r
                                       for one-byte V: see the kernel), over l >= 1
  scores and sums in fp32              2^-14 A (|s| log2(e) 2^-23 and the products'
                                       2^-24 sqrt(hd) |q| |k|, below 2^-15 at the
                                       scores of up to 60 used here)"""
import ctypes

import numpy as np
import pytest

import cuqwen_amd as cq
from tests.conftest import tiny_config
from tests.gpu_util import Pool
from tests.pages_util import DevicePool, Hip, ceil

pytestmark = pytest.mark.gpu
L = cq.lib
KVS = [cq.KV_FP16, cq.KV_INT8, cq.KV_FP8]


@pytest.fixture
def g():
    p = Pool()
    yield p
    p.close()


class Case:
    """A batch of forked sequences (one pool, shared pages first) or, with `apart`, a prefix in a pool of
    its own and tables that hold only the sequences' own tokens.  `pad`: entries of the tables behind those
    in use (of -1), as a server's tables have: long tables are worked through in two launches, short ones in one."""

    def __init__(self, g, seed, kv, heads, n_kv, hd, page, prefix, own, form="own", apart=False, layers=1, qscale=1.5, pad=1):
        rng = self.rng = np.random.default_rng(seed)
        self.g, self.kv, self.heads, self.n_kv, self.hd, self.page, self.prefix = g, kv, heads, n_kv, hd, page, prefix
        self.batch = len(own)
        self.layer = layers - 1
        full = 0 if apart else prefix // page
        self.start = 0 if apart else prefix
        self.lens = [n if n < 0 else self.start + n for n in own]
        more = [max(ceil(max(n, 0), page) - full, 0) for n in self.lens]
        n_pre = ceil(prefix, page)
        total = (0 if apart else full + (n_pre > full)) + sum(more) + 2
        ids = rng.permutation(total).tolist()
        shared, ids = ids[:full], ids[full:]
        self.rows = []
        for n in more:
            self.rows.append(shared + ids[:n])
            ids = ids[n:]
        self.pool = DevicePool(g, rng, kv, layers, total, page, n_kv, hd, form)
        if apart:
            self.pre = DevicePool(g, rng, kv, layers, n_pre + 1, page, n_kv, hd, "cache" if form == "own" else "own")
            self.pre_row = rng.permutation(n_pre + 1)[:n_pre].tolist()
        else:
            self.pre = self.pool
            self.pre_row = shared + ([ids[0]] if n_pre > full else [])
        self.width = max([len(r) for r in self.rows] + [1]) + pad
        self.pad = pad
        self.q = (rng.standard_normal((self.batch, heads, hd)) * qscale).astype(np.float16)

    def want(self):
        """(out, tolerance); NaN rows where nothing is written."""
        g, scale = self.heads // self.n_kv, 1 / np.sqrt(self.hd)
        out, tol = (np.full((self.batch, self.heads, self.hd), np.nan) for _ in range(2))
        pre = [self.pre.rows(k, self.layer, self.pre_row) if self.pre_row else np.zeros((0, self.n_kv, self.page, self.hd)) for k in (0, 1)]
        pre = [x.transpose(1, 0, 2, 3).reshape(self.n_kv, -1, self.hd)[:, :self.prefix] for x in pre]
        for b in range(self.batch):
            if self.lens[b] < 0:
                continue
            own = []
            for k in (0, 1):
                x = self.pool.rows(k, self.layer, self.rows[b]) if self.rows[b] else np.zeros((0, self.n_kv, self.page, self.hd))
                own.append(x.transpose(1, 0, 2, 3).reshape(self.n_kv, -1, self.hd)[:, self.start:max(self.lens[b], self.start)])
            for h in range(self.heads):
                K, V = (np.concatenate([pre[k][h // g], own[k][h // g]]) for k in (0, 1))
                if not len(K):
                    out[b, h] = tol[b, h] = 0
                    continue
                s = K @ self.q[b, h].astype(np.float64) * scale
                p = np.exp(s - s.max())
                w = p / p.sum()
                out[b, h] = w @ V
                top = np.abs(V).max() * 2   # r times the largest code: below twice the largest |v|
                tol[b, h] = 2.0 ** -11 * np.abs(out[b, h]) + 2.0 ** -25 + (2.0 ** -11 + 2.0 ** -14) * (w @ np.abs(V)) + \
                    2.0 ** -25 * top * len(K) / p.sum()
        return out, tol

    def put(self):
        g, n = self.g, self.heads * self.hd
        self.qs, self.os = n + 8, n + 24
        q = np.zeros((self.batch, self.qs), np.float16)
        q[:, :n] = self.q.reshape(self.batch, n)
        table = np.full((self.batch, self.width), -1, np.int32)
        for b, r in enumerate(self.rows):
            table[b, :len(r)] = r
        self.host_table = table
        self.d = dict(q=g.put(q), table=g.put(table), pre=g.i32(self.pre_row + [-1] * self.pad), plen=g.i32(self.prefix), start=g.i32(self.start),
                      lens=g.i32(self.lens))
        self.out = g.empty(self.batch * self.os * 2)
        self.ws = g.empty(L.cq_prefix_attention_workspace_bytes(self.batch, self.heads, self.n_kv, self.hd))
        return self

    def call(self, stream=None, start="start"):
        d = self.d
        cq.check(L.cq_prefix_attention_decode(d["q"], self.qs, self.out.ptr, self.os, self.pre.arg(), d["pre"], len(self.pre_row) + self.pad,
                                              d["plen"], self.pool.arg(), d["table"], self.width, d[start] if start else None, d["lens"],
                                              self.batch, self.layer, self.heads, self.ws.ptr, stream))

    def run(self):
        self.put()
        self.out.upload(np.full((self.batch, self.os), -9, np.float16))
        self.call(start="start" if self.start else None)
        return self.out.to_array(np.float16, (self.batch, self.os)).astype(np.float64)

    def check(self, got=None):
        got = self.run() if got is None else got
        n = self.heads * self.hd
        want, tol = (x.reshape(self.batch, n) for x in self.want())
        assert np.all(got[:, n:] == -9)
        gone = np.isnan(want)
        assert np.all(got[:, :n][gone] == -9)
        err = np.abs(got[:, :n] - want)[~gone]
        assert np.all(np.isfinite(got[:, :n])), "not finite"
        over = err - tol[~gone]
        assert err.size == 0 or over.max() <= 0, f"off by {err[over.argmax()]:.3g}, tolerance {tol[~gone][over.argmax()]:.3g}"


SHAPES = [(14, 2, 64), (28, 4, 128), (4, 4, 64), (16, 1, 128), (5, 5, 128), (40, 8, 128)]


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("heads,n_kv,hd", SHAPES)
def test_head_layouts(g, kv, heads, n_kv, hd):
    Case(g, heads, kv, heads, n_kv, hd, 64, 130, [1, 70, 33], layers=2).check()


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("heads,n_kv,hd", SHAPES)
def test_head_layouts_of_a_long_prefix(g, kv, heads, n_kv, hd):
    Case(g, heads + 1, kv, heads, n_kv, hd, 64, 2500, [1, 70, 33, 0], layers=2, pad=100).check()


@pytest.mark.parametrize("pad", [1, 300])
@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("page", [32, 64, 256])
@pytest.mark.parametrize("prefix", [0, 1, 31, 32, 33, 64, 255, 256, 257, 1000, 1792, 1793, 2047, 2048, 2049, 2177, 4000])
def test_prefix_lengths(g, kv, page, prefix, pad):
    Case(g, prefix + page, kv, 6, 2, 64, page, prefix, [0, 1, 31, 32, 65, -1, 300], pad=pad).check()


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("prefix", [0, 40, 2000])
@pytest.mark.parametrize("batch", [2, 40])
def test_own_lengths(g, kv, prefix, batch):
    """Around the own tiles that the second launch takes itself (16 or 64 of them) and past them."""
    own = [510, 512, 513, 544, 2047, 2048, 2049, 2080, 2500, 5000, 1, 0]
    own = own[:batch] if batch < 10 else own + [7] * (batch - len(own))
    Case(g, prefix + batch, kv, 6, 2, 64, 32, prefix, own, pad=40).check()
    Case(g, prefix + batch, kv, 5, 1, 128, 64, prefix, own[::-1], pad=40, apart=True).check()


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("form", ["own", "wide", "cache"])
def test_prefix_in_a_pool_of_its_own(g, kv, form):
    Case(g, 3, kv, 14, 2, 64, 64, 333, [0, 1, 100, 64, -5, 7], form, apart=True, layers=3).check()
    Case(g, 4, kv, 4, 2, 128, 32, 0, [0, 5, 64, -1], form, apart=True).check()


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("batch", [1, 2, 3, 5, 9, 10, 16, 19, 33, 37, 64, 74, 130])
def test_batches(g, kv, batch):
    rng = np.random.default_rng(batch)
    Case(g, batch, kv, 14, 2, 64, 32, 700, rng.integers(0, 90, batch).tolist()).check()
    Case(g, batch, kv, 7, 1, 128, 64, 999, rng.integers(0, 60, batch).tolist()).check()


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("batch", [1, 2, 3, 5, 9, 10, 16, 19, 33, 37, 64, 74, 130])
def test_batches_over_a_long_prefix(g, kv, batch):
    """Every number of rows per block of the first launch, rows that fill the last block or do not."""
    rng = np.random.default_rng(batch)
    Case(g, batch, kv, 14, 2, 64, 32, 3333, rng.integers(0, 90, batch).tolist()).check()
    Case(g, batch, kv, 7, 1, 128, 64, 5000, rng.integers(0, 60, batch).tolist()).check()


def test_largest_batch(g):
    rng = np.random.default_rng(1)
    Case(g, 3, cq.KV_FP8, 3, 1, 64, 64, 700, rng.integers(0, 40, 1024).tolist(), pad=1000).check()
    for heads, hd in ((16, 128), (9, 128), (16, 64), (8, 128)):
        Case(g, 4, cq.KV_INT8, heads, 1, hd, 64, 2100, rng.integers(0, 40, 270).tolist(), pad=100).check()
    Case(g, 1, cq.KV_FP16, 2, 1, 64, 32, 100, rng.integers(0, 40, 1024).tolist()).check()
    Case(g, 2, cq.KV_INT8, 2, 2, 64, 32, 2500, rng.integers(0, 40, 1023).tolist()).check()


@pytest.mark.parametrize("kv", KVS)
def test_long_prefix_and_ragged_own(g, kv):
    Case(g, 5, kv, 14, 2, 64, 128, 9001, [3000, 1, 0, 513, 64, 31, 2, 1999]).check()
    Case(g, 6, kv, 7, 1, 128, 64, 20011, [7] * 40).check()


@pytest.mark.parametrize("kv", KVS)
def test_only_own_tokens_or_nothing(g, kv):
    Case(g, 7, kv, 4, 2, 64, 32, 0, [0, 0, 0]).check()
    Case(g, 8, kv, 4, 2, 64, 32, 0, [5000, 0, 1]).check()
    Case(g, 9, kv, 4, 2, 64, 32, 0, [-1, -1]).check()
    Case(g, 10, kv, 4, 2, 64, 32, 77, [-1, -3]).check()


@pytest.mark.parametrize("kv", KVS)
def test_sharp_and_large_scores(g, kv):
    """Scores of some tens: the weights of one key or two decide.  Every form, since each keeps its running maximum."""
    for batch, prefix in ((3, 500), (2, 2500), (4, 2500), (9, 2500), (18, 2500), (30, 2500)):
        Case(g, 11, kv, 14, 2, 64, 64, prefix, ([20, 100, 3] * 10)[:batch], qscale=12).check()


@pytest.mark.parametrize("kv", [cq.KV_INT8, cq.KV_FP8])
@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -20, 2.0 ** 8])
@pytest.mark.parametrize("batch,prefix,hd", [(3, 400, 64), (3, 2300, 64), (12, 2300, 128), (40, 2300, 64), (40, 2300, 128)])
def test_small_and_large_scales_of_v(g, kv, size, batch, prefix, hd):
    """One-byte V whose scales would drive fp16 products into the subnormals, or rows of very different size."""
    c = Case(g, 12, kv, 7, 1, hd, 32, prefix, ([50, 3, 77] * 14)[:batch])
    for s in c.pool.scales[1:]:
        s *= np.float32(size) * np.where(c.rng.random(s.shape) < 0.5, 1, 2.0 ** -9).astype(np.float32)
    c.pool.upload()
    got = c.run()
    n = c.heads * c.hd
    want, tol = (x.reshape(c.batch, n) for x in c.want())
    assert np.all(np.abs(got[:, :n] - want) <= tol)


@pytest.mark.parametrize("kv", [cq.KV_INT8, cq.KV_FP8])
@pytest.mark.parametrize("share", [1.0, 0.5])
@pytest.mark.parametrize("batch,prefix", [(3, 400), (3, 2300), (12, 2300), (40, 2300)])
def test_scales_below_zero(g, kv, share, batch, prefix):
    """The store writes no such scale, but the formula takes it, all of them or some."""
    c = Case(g, 15, kv, 7, 1, 64, 32, prefix, ([50, 3, 77] * 14)[:batch])
    for s in c.pool.scales:
        s *= np.where(c.rng.random(s.shape) < share, -1, 1).astype(np.float32)
    c.pool.upload()
    got = c.run()
    n = c.heads * c.hd
    want, tol = (x.reshape(c.batch, n) for x in c.want())
    assert np.all(np.abs(got[:, :n] - want) <= tol)


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("what", [np.nan, np.inf, -65504.0])
@pytest.mark.parametrize("batch,prefix", [(5, 100), (2, 2500), (5, 2500), (12, 2501), (25, 2497)])
def test_anything_may_lie_behind_the_lengths(g, kv, what, batch, prefix):
    """Slots past a prefix and past a sequence, before its start, and pages that nobody names."""
    c = Case(g, 13, kv, 14, 2, 64, 64, prefix, ([20, 29, 1, 0, 64] * 5)[:batch])
    ref = c.want()
    seen = np.zeros((c.pool.n_pages, c.page), bool)
    for t in range(c.prefix):
        seen[c.pre_row[t // c.page], t % c.page] = True
    for row, n in zip(c.rows, c.lens):
        for t in range(c.start, n):
            seen[row[t // c.page], t % c.page] = True
    for k in (0, 1):
        for p, t in zip(*np.nonzero(~seen)):
            at = c.pool.at[0, p]
            for h in range(c.n_kv):
                o = at[h] + c.pool.offsets(k)[t]
                if kv == cq.KV_FP16:
                    c.pool.host[k][o] = what
                else:
                    c.pool.host[k][o] = 127 if kv == cq.KV_FP8 else -128   # E4M3: the NaN code
                    c.pool.scales[k][at[h] // c.hd + t] = what
    c.pool.upload()
    got = c.run()
    n = c.heads * c.hd
    want, tol = (x.reshape(c.batch, n) for x in ref)
    assert np.all(np.abs(got[:, :n] - want) <= tol)


@pytest.mark.parametrize("prefix", [64, 2560])
def test_infinities_and_nan_that_are_seen(g, prefix):
    """A NaN or an infinite score among the visible keys shows in the rows that see it, and only there."""
    c = Case(g, 14, cq.KV_FP16, 4, 2, 64, 32, prefix, [10, 12, 3])
    p, t = c.rows[1][prefix // 32], 3           # an own token of sequence 1, kv head 1
    c.pool.host[1][c.pool.at[0, p, 1] + c.pool.offsets(1)[t]] = np.nan
    c.pool.upload()
    got = c.run()[:, :c.heads * c.hd].reshape(c.batch, c.heads, c.hd)
    assert np.isnan(got[1, 2:]).all() and np.isfinite(got[1, :2]).all() and np.isfinite(got[[0, 2]]).all()
    c.pool.host[1][c.pool.at[0, p, 1] + c.pool.offsets(1)[t]] = 0
    c.pool.host[0][c.pool.at[0, c.pre_row[0], 0] + c.pool.offsets(0)[5]] = np.inf   # a prefix key of kv head 0: scores of +-inf or NaN
    c.pool.upload()
    got = c.run()[:, :c.heads * c.hd].reshape(c.batch, c.heads, c.hd)
    assert np.isnan(got[:, :2]).any(-1).all() and np.isfinite(got[:, 2:]).all()


def test_pages_outside_the_pool_are_not_seen(g):
    for batch, prefix, kv in ((3, 200, cq.KV_FP16), (40, 200, cq.KV_FP8), (2, 2600, cq.KV_INT8), (3, 2600, cq.KV_FP16), (12, 2600, cq.KV_FP8),
                              (12, 2600, cq.KV_FP16), (40, 2600, cq.KV_FP16), (40, 2600, cq.KV_INT8)):
        own = ([40, 70, 33] + [20] * batch)[:batch]
        c = Case(g, 15, kv, 14, 2, 64, 32, prefix, own)
        c.put()
        table = c.host_table.copy()
        first = prefix // 32                                    # the page of the first own token
        table[1, first + 1], table[0, first] = c.pool.n_pages, -2 ** 31
        pre = list(c.pre_row)
        pre[2], pre[4] = 2 ** 31 - 1, -1                        # prefix positions 64..95, 128..159
        c.d["table"], c.d["pre"] = g.put(table), g.i32(pre + [-1])
        c.out.upload(np.full((c.batch, c.os), -9, np.float16))
        c.call()
        got = c.out.to_array(np.float16, (c.batch, c.os)).astype(np.float64)[:, :c.heads * c.hd]
        scale, grp = 1 / np.sqrt(c.hd), c.heads // c.n_kv
        for b in range(min(3, batch)):
            for h in range(c.heads):
                K = []
                for t in range(c.prefix):
                    if t // 32 not in (2, 4):
                        K.append((c.pre_row[t // 32], t % 32))
                for t in range(c.prefix, c.lens[b]):
                    if not (b == 1 and t // 32 == first + 1) and not (b == 0 and t // 32 == first):
                        K.append((c.rows[b][t // 32], t % 32))
                pid, tok = (np.array(x) for x in zip(*K))
                k, v = (c.pool.rows(i, 0, pid)[np.arange(len(pid)), h // grp, tok] for i in (0, 1))
                s = k @ c.q[b, h].astype(np.float64) * scale
                p = np.exp(s - s.max())
                w = p / p.sum()
                tol = 2.0 ** -11 * np.abs(w @ v) + 2.0 ** -24 + (2.0 ** -11 + 2.0 ** -14) * (w @ np.abs(v)) + \
                    2.0 ** -24 * np.abs(v).max() * len(k) / p.sum()
                assert np.all(np.abs(got[b, h * c.hd:(h + 1) * c.hd] - w @ v) <= tol), (batch, b, h)


def test_lengths_are_cut_at_the_tables(g):
    """A prefix length, a sequence length and a start past what the tables hold, or below zero."""
    c = Case(g, 16, cq.KV_INT8, 4, 2, 64, 32, 96, [10, 20, 32])
    ref = c.run()
    c.d["plen"] = g.i32(-4)
    c.d["start"] = g.i32(-7)          # everything from position 0 on, by each sequence's own table
    c.call()
    got = c.out.to_array(np.float16, (c.batch, c.os)).astype(np.float64)
    want, tol = c.want()
    n = c.heads * c.hd
    assert np.all(np.abs(got[:, :n] - want.reshape(c.batch, n)) <= tol.reshape(c.batch, n))
    assert np.all(np.abs(ref[:, :n] - want.reshape(c.batch, n)) <= tol.reshape(c.batch, n))
    c = Case(g, 17, cq.KV_FP16, 4, 2, 64, 32, 96, [32, 32], apart=True)
    c.put()
    c.d["plen"], c.d["lens"] = g.i32(2 ** 31 - 1), g.i32([2 ** 31 - 1, 2 ** 31 - 1])
    c.out.upload(np.full((c.batch, c.os), -9, np.float16))
    c.call(start=None)                # the entries behind are -1: nothing there is seen
    c.check(c.out.to_array(np.float16, (c.batch, c.os)).astype(np.float64))
    c.d["start"] = g.i32(2 ** 31 - 1)
    c.call()                          # no own position left
    c.lens = [0, 0]
    c.check(c.out.to_array(np.float16, (c.batch, c.os)).astype(np.float64))


@pytest.mark.parametrize("prefix,batch", [(500, 40), (2900, 3), (2900, 12), (2900, 40)])
def test_same_bits_on_every_call(g, prefix, batch):
    """Fixed order of all sums: two calls, and a call with a workspace full of NaN, agree bit for bit."""
    c = Case(g, 18, cq.KV_FP16, 28, 4, 128, 64, prefix, ([100, 3, 0, 40, 77] * 8)[:batch])
    a = c.run()
    c.ws.upload(np.full(c.ws.nbytes // 2, np.nan, np.float16))
    c.call(start="start")
    b = c.out.to_array(np.float16, (c.batch, c.os)).astype(np.float64)
    assert np.array_equal(a, b)
    c.check(b)


@pytest.mark.parametrize("kv", KVS)
@pytest.mark.parametrize("prefix", [300, 2700])
def test_captured_with_growing_lengths(g, kv, prefix):
    """One graph, replayed as the sequences grow; eager calls of the same state between the replays."""
    c = Case(g, 19, kv, 14, 2, 64, 64, prefix, [200, 40, 90, 33, 64, 1], pad=100)
    c.put()
    c.out.upload(np.full((c.batch, c.os), -9, np.float16))
    hip = Hip()
    stream = hip.stream()
    cq.synchronize()
    graph = hip.capture(stream, lambda: c.call(stream))
    full = list(c.lens)
    for cut in (190, 100, 0, 33):
        c.lens = [max(n - cut, c.start) for n in full]
        new = np.array(c.lens, np.int32)
        cq.check(L.cq_memcpy_h2d(c.d["lens"], new.ctypes.data, new.nbytes))
        hip.launch(graph, stream)
        hip.wait(stream)
        got = c.out.to_array(np.float16, (c.batch, c.os)).astype(np.float64)
        c.check(got)
        c.out.upload(np.full((c.batch, c.os), -9, np.float16))
        c.call()
        assert np.array_equal(c.out.to_array(np.float16, (c.batch, c.os)).astype(np.float64), got)
    hip.drop(stream, [graph])


def test_two_streams_with_workspaces_of_their_own(g):
    hip = Hip()
    streams = [hip.stream(), hip.stream()]
    cases = [Case(g, 20 + i, cq.KV_FP16, 14, 2, 64, 32, 2500 + i, [9, 70, 3, 40 + i]).put() for i in range(2)]
    for c in cases:
        c.out.upload(np.full((c.batch, c.os), -9, np.float16))
    cq.synchronize()
    for _ in range(5):
        for c, s in zip(cases, streams):
            c.call(s)
    for s in streams:
        hip.wait(s)
    for c in cases:
        c.check(c.out.to_array(np.float16, (c.batch, c.os)).astype(np.float64))
    for s in streams:
        hip.drop(s)


def test_prefix_is_a_states_own_cache(g):
    """The prompt that cq_prefill left in a state, read in place as the prefix of a batch."""
    cfg = tiny_config(max_seq_len=544)
    for kv in KVS:
        w = cq.synth_weights(cfg, 5)
        st = cq.State(cfg, w, kv_dtype=kv)
        st.prefill(list(range(1, 152)))
        c = Case(g, 22, kv, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, 32, 160, [5, 40, 0, 32], apart=True, layers=2)
        view = st.kv_pages(32)

        class View:   # the prefix's values as the state gives them out
            page_ids = None

            def arg(self):
                return ctypes.byref(view)

            def rows(self, kind, layer, ids):
                x = np.stack([st.kv_read(layer, h, kind, 160) for h in range(cfg.n_kv_heads)]).astype(np.float64)
                return x.reshape(cfg.n_kv_heads, 5, 32, cfg.head_dim).transpose(1, 0, 2, 3)[ids]

        c.pre, c.pre_row, c.prefix = View(), [0, 1, 2, 3, 4], 151
        if kv == cq.KV_FP16:
            c.check()
        else:   # kv_read rounds value * scale to fp16: 2^-11 of each key's products and of each v
            got = c.run()[:, :c.heads * c.hd]
            want, tol = (x.reshape(c.batch, -1) for x in c.want())
            k = np.abs(np.stack([c.pre.rows(0, 1, [0, 1, 2, 3, 4])])).max()
            slack = 2.0 ** -11 * (1 + 2 * k * np.abs(c.q).sum(-1).max() / np.sqrt(c.hd))
            assert np.all(np.abs(got - want) <= tol + slack * np.abs(c.pre.rows(1, 1, [0, 1, 2, 3, 4])).max())
        st.free()
        w.free()


@pytest.mark.parametrize("kv", KVS)
def test_offsets_past_32_bits(g, kv):
    """Pages whose elements lie past 2^32 of the pool's first: every step gives the bits that it gives in a small pool."""
    heads, n_kv, hd, page, prefix, own = 6, 2, 64, 32768, 3000, 70
    rng = np.random.default_rng(16)
    n = prefix + 2 * own
    rows = [(rng.standard_normal((n, n_kv * hd))).astype(np.float16) for _ in range(2)]
    q = g.put((rng.standard_normal((2, heads * hd)) * 1.5).astype(np.float16))
    got = []
    for ids, n_pages in (((0, 1, 2, 3), 4), ((1040, 1099, 3, 1057), 1100)):
        d = cq.kv_pages(page, n_kv, hd, n_pages, 1, kv)
        size, scales = cq.kv_pages_bytes(d)
        d.k, d.v = (g.empty(size).value for _ in range(2))
        if scales:
            d.k_scale, d.v_scale = (g.empty(scales).value for _ in range(2))
        pool = ctypes.byref(d)
        slots = [ids[0] * page + t for t in range(prefix)] + [i * page + t for i in ids[1:3] for t in range(own)]
        cq.check(L.cq_paged_kv_store(pool, 0, g.put(rows[0]), g.put(rows[1]), n_kv * hd, g.i32(slots), n, None))
        status = g.empty(4)
        cq.check(L.cq_pages_copy(pool, pool, g.i32([ids[1]]), g.i32([ids[3]]), 1, status.ptr, None))   # the first one's own page
        assert status.to_array(np.int32, (1,))[0] == 0
        out, ws = g.empty(2 * heads * hd * 2), g.empty(L.cq_prefix_attention_workspace_bytes(2, heads, n_kv, hd))
        cq.check(L.cq_prefix_attention_decode(q, heads * hd, out.ptr, heads * hd, pool, g.i32([ids[0]]), 1, g.i32([prefix]), pool,
                                              g.i32([ids[3], ids[2]]), 1, None, g.i32([own, own]), 2, 0, heads, ws.ptr, None))
        back = [g.empty(n * n_kv * hd * 2) for _ in range(2)]
        cq.check(L.cq_paged_kv_load(pool, 0, back[0].ptr, back[1].ptr, n_kv * hd, g.i32(slots), n, None))
        got.append([x.to_array(np.uint16, (x_n,)) for x, x_n in ((out, 2 * heads * hd), (back[0], n * n_kv * hd), (back[1], n * n_kv * hd))])
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    if kv == cq.KV_FP16:
        assert np.array_equal(got[0][1], rows[0].view(np.uint16).ravel()) and np.array_equal(got[0][2], rows[1].view(np.uint16).ravel())
    assert np.any(got[0][0])
