"""A paged KV cache kept by hand (numpy), its device counterpart, and the few HIP
runtime calls (streams, graph capture) that its tests need."""
import ctypes
import glob

import numpy as np

import cuqwen_amd as cq
from tests.gpu_util import k8_offsets, k_offsets, v8_offsets, v_offsets

OK, EINVAL, ENOMEM, ERANGE = 0, 1, 5, 6
INT_MAX = 2 ** 31 - 1


def ceil(a, b):
    return -(-a // b)


class Book:
    """The page map, one sequence and one token at a time."""

    def __init__(self, n_pages, n_seqs, max_pages, page):
        self.ref, self.len = [0] * n_pages, [0] * n_seqs
        self.table = [[-1] * max_pages for _ in range(n_seqs)]
        self.n_pages, self.n_seqs, self.max_pages, self.page = n_pages, n_seqs, max_pages, page

    def held(self, s):
        return ceil(self.len[s], self.page)

    def fork(self, parents, children):
        status = []
        for i, (p, c) in enumerate(zip(parents, children)):
            if not (0 <= p < self.n_seqs and 0 <= c < self.n_seqs):
                status.append(ERANGE)
            elif p in children or c in children[:i]:
                status.append(EINVAL)
            else:
                status.append(None)
        before = list(self.len)
        for i, (p, c) in enumerate(zip(parents, children)):
            if status[i] is not None:
                continue
            if before[c] != 0:
                status[i] = EINVAL
            elif not 0 <= before[p] <= self.max_pages * self.page:
                status[i] = ERANGE
            else:
                status[i] = OK
                self.len[c] = before[p]
                for k in range(self.held(p)):
                    q = self.table[c][k] = self.table[p][k]
                    if 0 <= q < self.n_pages:
                        self.ref[q] += 1
        return status

    def trim(self, seqs, keep=None):
        status = []
        for i, s in enumerate(seqs):
            want = keep[i] if keep is not None else 0
            if not 0 <= s < self.n_seqs or want < 0:
                status.append(ERANGE)
            elif s in seqs[:i]:
                status.append(EINVAL)
            elif not 0 <= self.len[s] <= self.max_pages * self.page:
                status.append(ERANGE)
            else:
                status.append(OK)
                if want < self.len[s]:
                    for k in range(ceil(want, self.page), self.held(s)):
                        q, self.table[s][k] = self.table[s][k], -1
                        if 0 <= q < self.n_pages:
                            self.ref[q] -= 1
                    self.len[s] = want
        return status

    def append(self, add, n_slots):
        """(slots, status, [(from, to, tokens)])"""
        none = [-1] * n_slots
        for s, a in enumerate(add):
            n = self.len[s]
            if a < 0 or n < 0 or n + a > self.max_pages * self.page:
                return none, [ERANGE, 0, 0, 0], []
            if a > 0 and n % self.page and not 0 <= self.table[s][self.held(s) - 1] < self.n_pages:
                return none, [ERANGE, 0, 0, 0], []
        if sum(add) > n_slots:
            return none, [ERANGE, 0, 0, 0], []
        ref, table = list(self.ref), [list(r) for r in self.table]
        free = [p for p in range(self.n_pages) if ref[p] <= 0]
        slots, moves, taken = [], [], 0
        for s, a in enumerate(add):
            n = self.len[s]
            fresh = []
            if a > 0 and n % self.page and ref[table[s][self.held(s) - 1]] > 1:
                fresh.append(self.held(s) - 1)
            copies = len(fresh)
            fresh += range(self.held(s), ceil(n + a, self.page))
            for k in fresh:
                p = free[taken] if taken < len(free) else None
                taken += 1
                if copies and k == fresh[0]:
                    ref[table[s][k]] -= 1
                    moves.append((table[s][k], p, ceil(n % self.page, 32) * 32))
                if p is not None:
                    table[s][k], ref[p] = p, 1
            if taken <= len(free):
                slots += [table[s][t // self.page] * self.page + t % self.page for t in range(n, n + a)]
        if taken > len(free):
            return none, [ENOMEM, taken, len(moves), sum(add)], []
        self.ref, self.table = ref, table
        self.len = [n + a for n, a in zip(self.len, add)]
        return slots + [-1] * (n_slots - len(slots)), [OK, taken, len(moves), sum(add)], moves

    def compact(self):
        """(remap, status, [(from, to)])"""
        used = [p for p in range(self.n_pages) if self.ref[p] > 0]
        holes = [p for p in range(len(used)) if self.ref[p] <= 0]
        moved = [p for p in used if p >= len(used)]
        remap = [p if self.ref[p] > 0 else -1 for p in range(self.n_pages)]
        for a, b in zip(moved, holes):
            remap[a], self.ref[b], self.ref[a] = b, self.ref[a], 0
        for s in range(self.n_seqs):
            for k in range(min(max(self.held(s), 0), self.max_pages)):
                p = self.table[s][k]
                if 0 <= p < self.n_pages and remap[p] >= 0:
                    self.table[s][k] = remap[p]
        return remap, [OK, len(used), len(moved), 0], list(zip(moved, holes))


class DeviceMap:
    def __init__(self, pool, book):
        self.book, self.n = book, (book.n_pages, book.n_seqs, book.max_pages, book.page)
        self.ref, self.table, self.len = (pool.empty(4 * n) for n in (book.n_pages, book.n_seqs * book.max_pages, book.n_seqs))
        self.desc = cq.page_map(self.ref.value, self.table.value, self.len.value, *self.n)
        self.upload()
        self.work = pool.empty(cq.lib.cq_pages_workspace_bytes(self.arg()))

    def arg(self):
        return ctypes.byref(self.desc)

    def upload(self):
        self.ref.upload(np.array(self.book.ref, np.int32))
        self.table.upload(np.array(self.book.table, np.int32))
        self.len.upload(np.array(self.book.len, np.int32))

    def same(self):
        b = self.book
        assert np.array_equal(self.len.to_array(np.int32), np.array(b.len)), "len"
        assert np.array_equal(self.ref.to_array(np.int32), np.array(b.ref)), "ref"
        assert np.array_equal(self.table.to_array(np.int32, (b.n_seqs, b.max_pages)), np.array(b.table)), "table"


class DevicePool:
    """Random bytes in the shape of a pool; `form` "own" (pages one behind the other),
    "cache" (as in a state: head after head) or "wide" (gaps between heads, pages, layers)."""

    def __init__(self, pool, rng, kv, layers, n_pages, page, n_kv, hd, form="own"):
        self.kv, self.layers, self.n_pages, self.page, self.n_kv, self.hd = kv, layers, n_pages, page, n_kv, hd
        run, es = page * hd, 2 if kv == cq.KV_FP16 else 1
        if form == "cache":
            s = (n_kv * (n_pages * run + 32 * hd), run, n_pages * run + 32 * hd)
        elif form == "wide":
            s = (n_pages * (n_kv * (run + 32 * hd) + 64 * hd) + 32 * hd, n_kv * (run + 32 * hd) + 64 * hd, run + 32 * hd)
        else:
            s = (n_pages * n_kv * run, n_kv * run, run)
        self.strides, elems = s, layers * s[0]
        # element offset of (layer, page, head)
        self.at = (np.arange(layers)[:, None, None] * s[0] + np.arange(n_pages)[:, None] * s[1] + np.arange(n_kv) * s[2]).astype(np.int64)
        self.host = [self._random(rng, elems, es) for _ in range(2)]
        self.scales = None if es == 2 else [np.exp(rng.standard_normal(elems // hd) * 0.3).astype(np.float32) / 50 for _ in range(2)]
        self.dev = [pool.empty(x.nbytes) for x in self.host]
        self.sdev = None if self.scales is None else [pool.empty(x.nbytes) for x in self.scales]
        self.desc = cq.kv_pages(page, n_kv, hd, n_pages, layers, kv, self.dev[0].value, self.dev[1].value,
                                self.sdev[0].value if self.sdev else None, self.sdev[1].value if self.sdev else None)
        self.desc.layer_stride, self.desc.page_stride, self.desc.head_stride = s
        self.upload()

    def _random(self, rng, n, es):
        if es == 2:
            return rng.standard_normal(n).astype(np.float16)
        if self.kv == cq.KV_INT8:
            return rng.integers(-127, 128, n, dtype=np.int8)
        c = rng.integers(0, 127, n, dtype=np.uint8) | (rng.integers(0, 2, n, dtype=np.uint8) << 7)   # no NaN code
        return c.view(np.int8)

    def arg(self):
        return ctypes.byref(self.desc)

    def upload(self):
        for d, h in zip(self.dev + (self.sdev or []), self.host + (self.scales or [])):
            d.upload(h)

    def _move(self, a, b, tokens, other=None):
        src = other or self
        for k in range(2):
            for l in range(self.layers):
                for h in range(self.n_kv):
                    x, y = src.at[l, a, h], self.at[l, b, h]
                    n = tokens * self.hd
                    self.host[k][y:y + n] = src.host[k][x:x + n]
                    if self.scales:
                        self.scales[k][y // self.hd:y // self.hd + tokens] = src.scales[k][x // self.hd:x // self.hd + tokens]

    def move(self, pairs):
        for p in pairs:
            self._move(p[0], p[1], p[2] if len(p) > 2 else self.page)

    def same(self):
        for d, h in zip(self.dev + (self.sdev or []), self.host + (self.scales or [])):
            got = d.to_array(h.dtype)
            assert np.array_equal(got.view(np.uint8), h.view(np.uint8)), "pool"

    def offsets(self, kind):
        """In-page element offsets [page token][hd]."""
        f = ((k_offsets, v_offsets) if self.kv == cq.KV_FP16 else (k8_offsets, v8_offsets))[kind]
        return f(1, self.page, self.hd, self.page)[0]

    def rows(self, kind, layer, page_ids):
        """[page][head][token][hd] values in 64 bits."""
        at = self.at[layer, page_ids][..., None, None] + self.offsets(kind)
        x = values(self.host[kind][at], self.kv)
        if self.scales is None:
            return x
        s = self.scales[kind][self.at[layer, page_ids][..., None] // self.hd + np.arange(self.page)]
        return x * s.astype(np.float64)[..., None]


def values(codes, kv):
    if kv == cq.KV_FP16 or kv == cq.KV_INT8:
        return codes.astype(np.float64)
    c = codes.view(np.uint8).astype(np.int64)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    a = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * np.exp2(np.maximum(e, 1) - 7.0))
    a = np.where((c & 127) == 127, np.nan, a)
    return np.where(c >= 128, -a, a)


class Hip:
    """Streams and graph capture of the runtime that the library uses."""

    def __init__(self):
        self.lib = ctypes.CDLL(glob.glob("/opt/rocm/lib/libamdhip64.so.[0-9]")[0])

    def __call__(self, name, *args):
        rc = getattr(self.lib, name)(*args)
        assert rc == 0, f"{name}: {rc}"

    def stream(self):
        s = ctypes.c_void_p()
        self("hipStreamCreateWithFlags", ctypes.byref(s), 1)   # non-blocking
        return s

    def capture(self, stream, body):
        g, e = ctypes.c_void_p(), ctypes.c_void_p()
        self("hipStreamBeginCapture", stream, 1)   # thread local
        try:
            body()
        finally:
            self("hipStreamEndCapture", stream, ctypes.byref(g))
        self("hipGraphInstantiate", ctypes.byref(e), g, None, None, ctypes.c_size_t(0))
        self("hipGraphDestroy", g)
        return e

    def launch(self, graph, stream):
        self("hipGraphLaunch", graph, stream)

    def wait(self, stream):
        self("hipStreamSynchronize", stream)

    def drop(self, stream=None, graphs=()):
        for e in graphs:
            self("hipGraphExecDestroy", e)
        if stream is not None:
            self("hipStreamDestroy", stream)
