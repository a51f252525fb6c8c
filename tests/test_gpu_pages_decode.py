"""GPU test of the paged operators together, as a program uses them for several answers
to one prompt: the prompt prefilled once in a state, its pages copied into a pool, forked
for the answers, and decode steps of the batch through the op-level entry points (page
append, row store, attention over the shared prefix) -- against a state of its own for
each answer.  Midway one answer ends and the pool is compacted."""
import ctypes

import numpy as np
import pytest

import cuqwen_amd as cq
from tests.conftest import tiny_config
from tests.gpu_util import Pool, rel_err
from tests.pages_util import Book, DeviceMap, DevicePool, ceil

pytestmark = pytest.mark.gpu
L = cq.lib
TOL = 1e-2   # as the decode step against the oracle: other orders of the same sums, scores not rounded to fp16 here


class Batch:
    """Rows of a batch through one model's layers, by the op-level calls."""

    def __init__(self, g, cfg, w, n):
        self.g, self.c, self.w, self.n = g, cfg, w, n
        qd, kvd = cfg.n_heads * cfg.head_dim, cfg.n_kv_heads * cfg.head_dim
        self.qd, self.kvd, self.row = qd, kvd, qd + 2 * kvd
        self.x, self.h, self.qkv, self.att = (g.empty(2 * n * k) for k in (cfg.dim, cfg.dim, self.row, qd))
        self.inter, self.logits = g.empty(2 * cfg.intermediate_size), g.empty(2 * cfg.vocab_size)
        self.wo = []
        for l in range(cfg.n_layers):
            a, b = ctypes.c_void_p(), ctypes.c_void_p()
            cq.check(L.cq_weights_wo_rows(w.handle, l, ctypes.byref(a), ctypes.byref(b)))
            self.wo.append((a, b))

    def t(self, name, layer=-1):
        return self.w.tensor(name, layer)[0]

    def step(self, tokens, positions, kv, slots, attend):
        """One token of each row: store(layer) by slots, attend(layer, q, q_stride, out, out_stride)."""
        c, g, q8 = self.c, self.g, self.c.quant_type
        pos = [g.i32(p) for p in positions]
        for b, tok in enumerate(tokens):
            cq.check(L.cq_embedding_lookup(self.t("embed"), g.i32(tok), self.x.value + 2 * b * c.dim, c.dim, None))
        for l in range(c.n_layers):
            for b in range(self.n):
                at = self.qkv.value + 2 * b * self.row
                cq.check(L.cq_fused_attn_block(
                    q8, self.x.value + 2 * b * c.dim, self.t("in_norm", l), self.t("wq", l), self.t("wk", l), self.t("wv", l),
                    self.t("sq", l), self.t("sk", l), self.t("sv", l), self.t("bq", l), self.t("bk", l), self.t("bv", l), at,
                    at + 2 * self.qd, at + 2 * (self.qd + self.kvd), c.dim, c.n_heads, c.n_kv_heads, c.head_dim, pos[b], c.rope_theta,
                    c.norm_eps, None))
            cq.check(L.cq_paged_kv_store(kv, l, self.qkv.value + 2 * self.qd, self.qkv.value + 2 * (self.qd + self.kvd), self.row, slots,
                                         self.n, None))
            attend(l, self.qkv.value, self.row, self.att.value, self.qd)
            for b in range(self.n):
                x = self.x.value + 2 * b * c.dim
                cq.check(L.cq_gemv_add(q8, self.wo[l][0], self.wo[l][1], self.att.value + 2 * b * self.qd, x, c.dim, self.qd, None))
                cq.check(L.cq_fused_mlp_stage1(q8, x, self.t("post_norm", l), self.t("wg", l), self.t("wu", l), self.t("sg", l),
                                               self.t("su", l), self.inter.ptr, c.dim, c.intermediate_size, c.norm_eps, None))
                cq.check(L.cq_fused_mlp_stage2(q8, x, self.t("wd", l), self.t("sd", l), self.inter.ptr, c.dim, c.intermediate_size, None))
        out = []
        for b in range(self.n):
            cq.check(L.cq_rmsnorm(self.x.value + 2 * b * c.dim, self.t("final_norm"), self.h.ptr, c.dim, c.norm_eps, None))
            cq.check(L.cq_compute_logits(c.lm_head_fmt, self.h.ptr, self.t("lm_head"), None, self.logits.ptr, c.vocab_size, c.dim, None))
            out.append(self.logits.to_array(np.float16).astype(np.float64))
        return out


@pytest.mark.parametrize("kv", [cq.KV_FP16, cq.KV_INT8, cq.KV_FP8])
@pytest.mark.parametrize("prompt,page,shared", [(75, 32, "pool"), (96, 32, "pool"), (75, 64, "state"), (1, 32, "pool")])
def test_answers_to_one_prompt(kv, prompt, page, shared):
    """`shared` "pool": the prompt's pages in the pool, forked; "state": read in place in the state's own cache."""
    g = Pool()
    cfg = tiny_config(repetition_penalty=1.0)
    w = cq.synth_weights(cfg, 31)
    rng = np.random.default_rng(prompt + page)
    text = rng.integers(0, cfg.vocab_size, prompt).tolist()
    n = 4
    st = cq.State(cfg, w, kv_dtype=kv)
    refs = [cq.State(cfg, w, kv_dtype=kv) for _ in range(n)]
    for s in [st] + refs:
        s.prefill(text)
    pool = DevicePool(g, rng, kv, cfg.n_layers, 40, page, cfg.n_kv_heads, cfg.head_dim)
    view = st.kv_pages(page)
    book = Book(40, n + 1, 8, page)
    m = DeviceMap(g, book)
    slots, status = g.empty(4 * max(prompt, n)), g.empty(16)

    def append(add, total):
        cq.check(L.cq_pages_append(pool.arg(), m.arg(), g.i32(add), slots.ptr, total, status.ptr, m.work.ptr, None))
        assert status.to_array(np.int32)[0] == 0 and status.to_array(np.int32)[3] == sum(add)

    if shared == "pool":
        append([prompt] + [0] * n, prompt)
        row = m.table.to_array(np.int32, (n + 1, 8))[0, :ceil(prompt, page)]
        cq.check(L.cq_pages_copy(ctypes.byref(view), pool.arg(), g.i32(range(len(row))), g.i32(row), len(row), g.empty(4 * len(row)).ptr, None))
        st4 = g.empty(4 * n)
        cq.check(L.cq_pages_fork(m.arg(), g.i32([0] * n), g.i32(list(range(1, n + 1))), n, st4.ptr, None))
        assert not st4.to_array(np.int32).any()
    batch = Batch(g, cfg, w, n)
    ws = g.empty(L.cq_prefix_attention_workspace_bytes(n, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim))
    plen, zero = g.i32(prompt), g.i32(0)
    table, lens = m.table.value + 4 * 8, m.len.value + 4          # rows of the answers

    def attend(l, q, qs, out, os):
        if shared == "pool":
            args = (pool.arg(), m.table.ptr, 8, plen, pool.arg(), table, 8, plen, lens)
        else:
            args = (ctypes.byref(view), g.i32(range(view.n_pages)), view.n_pages, plen, pool.arg(), table, 8, zero, lens)
        cq.check(L.cq_prefix_attention_decode(q, qs, out, os, *args, n, l, cfg.n_heads, ws.ptr, None))

    for step in range(40):
        tokens = rng.integers(0, cfg.vocab_size, n).tolist()
        append([0] + [1] * n, n)
        got = batch.step(tokens, [prompt + step] * n, pool.arg(), slots.ptr, attend)
        for b in range(n):
            refs[b].forward(tokens[b], prompt + step)
            want = refs[b].logits().astype(np.float64)
            assert rel_err(got[b], want) <= TOL, (step, b)
        if step == 20:   # the prompt's own entry ends (its pages stay with the answers), the pool moves together
            if shared == "pool":
                cq.check(L.cq_pages_trim(m.arg(), zero, None, 1, status.ptr, None))
                m_rows = m.table.to_array(np.int32, (n + 1, 8))
                assert m_rows[0].max() == -1
                remap = g.empty(4 * 40)
                cq.check(L.cq_pages_compact(pool.arg(), m.arg(), remap.ptr, status.ptr, m.work.ptr, None))
                used = status.to_array(np.int32)[1]
                assert m.table.to_array(np.int32, (n + 1, 8)).max() < used

                def attend(l, q, qs, out, os):   # the prefix by the first answer's row from here on
                    cq.check(L.cq_prefix_attention_decode(q, qs, out, os, pool.arg(), table, 8, plen, pool.arg(), table, 8, plen, lens, n,
                                                          l, cfg.n_heads, ws.ptr, None))
    for s in [st] + refs:
        s.free()
    w.free()
    g.close()
