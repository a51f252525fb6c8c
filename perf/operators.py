"""Timed cases of the paged KV cache: a batch of answers that share one prompt.

The K and V of every layer live in pages of `page` tokens (each page holds all
kv heads, in the tile order of the engine's own cache), tables name the pages
of each sequence, and a page named by several tables is stored once.

Kinds of case:
  attn     decode attention of one layer for a batch whose sequences share a
           prompt and have their own tokens behind it
  store    rows of new K and V into pages; a one-byte cache is read back too,
           as the values that its codes stand for
  copy     the pages of a prompt that a contiguous cache holds, into the pool
  branch   the last answers' pages given back, the prompt forked for the next
           ones, and room for each one's first token (the partly filled last
           page of the prompt is copied for each)
  compact  half of the sequences end, the pages move together, and new
           sequences take the room behind them
"""
import ctypes
import math

import torch

own = False

DEV = "cuda"
MODELS = {"0.5B": (14, 2, 64), "1.5B": (12, 2, 128), "3B": (16, 2, 128), "7B": (28, 4, 128), "14B": (40, 8, 128)}
KV_TAG = {"fp16": 0, "int8": 1, "fp8": 2}


def listed():
    return [
        # two answers to a one-line question: launch bound
        dict(name="attn-0.5B-2x100", kind="attn", model="0.5B", kv="fp16", page=32, batch=2, prefix=100, most=20),
        # 64 samples of one long document's summary, some hundred tokens in
        dict(name="attn-7B-64x32k", kind="attn", model="7B", kv="fp16", page=64, batch=64, prefix=32640, most=1000),
        # a few answers over an E4M3 cache
        dict(name="attn-14B-8x20k-fp8", kind="attn", model="14B", kv="fp8", page=128, batch=8, prefix=20001, most=700),
        # ragged int8: an odd batch, a prompt that ends inside a page
        dict(name="attn-0.5B-33x3001-int8", kind="attn", model="0.5B", kv="int8", page=32, batch=33, prefix=3001, most=333),
        # one step's rows of a batch; a chunk of a prompt
        dict(name="store-7B-64-int8", kind="store", model="7B", kv="int8", page=64, tokens=64, chunk=1),
        dict(name="store-1.5B-2048", kind="store", model="1.5B", kv="fp16", page=64, tokens=2048, chunk=2048),
        # a prompt out of the engine's own cache, all layers; a long one of a few layers
        dict(name="copy-0.5B-2k", kind="copy", model="0.5B", kv="fp16", page=32, layers=24, tokens=2000),
        dict(name="copy-7B-32k-int8", kind="copy", model="7B", kv="int8", page=128, layers=6, tokens=32768),
        # four answers to a short question; 64 to a long one
        dict(name="branch-0.5B-4x300", kind="branch", model="0.5B", kv="fp16", page=32, layers=24, prompt=300, children=4),
        dict(name="branch-7B-64x20k", kind="branch", model="7B", kv="fp16", page=64, layers=8, prompt=20011, children=64),
        # a small pool, and a pool of a busy server's size in pages
        dict(name="compact-1.5B-16", kind="compact", model="1.5B", kv="fp8", page=32, layers=28, seqs=16, most=300),
        dict(name="compact-7B-96", kind="compact", model="7B", kv="fp16", page=64, layers=6, seqs=96, most=1500),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["attn", "attn", "attn", "store", "copy", "branch", "compact"])
    model, kv, page = rng.choice(list(MODELS)), rng.choice(["fp16", "fp16", "int8", "fp8"]), rng.choice([32, 64, 128])
    heads, n_kv, hd = MODELS[model]
    c = dict(kind=kind, model=model, kv=kv, page=page)
    if kind == "attn":
        batch = _log_int(rng, 1, 256)
        # no more products than the largest listed case, no more own tokens
        prefix = _log_int(rng, 1, max(1, min(32768, int(7e9 / (batch * heads * hd)))))
        return dict(c, batch=batch, prefix=prefix, most=_log_int(rng, 1, max(1, min(1200, int(1.6e7 / (batch * n_kv * hd))))))
    if kind == "store":
        chunk = rng.choice([1, 1, _log_int(rng, 2, 2048)])
        return dict(c, tokens=_log_int(rng, 1, 256) if chunk == 1 else max(chunk, _log_int(rng, 2, 4096)), chunk=chunk)
    if kind == "copy":
        layers = _log_int(rng, 2, 24)
        return dict(c, layers=layers, tokens=_log_int(rng, 1, int(8e7 / (layers * n_kv * hd))))
    if kind == "branch":
        layers = _log_int(rng, 2, 16)
        return dict(c, layers=layers, prompt=_log_int(rng, 1, int(8e7 / (layers * n_kv * hd))), children=_log_int(rng, 1, 96))
    layers, seqs = _log_int(rng, 2, 16), _log_int(rng, 2, 128)
    return dict(c, layers=layers, seqs=seqs, most=_log_int(rng, 2, max(2, min(2000, int(1.2e8 / (layers * n_kv * hd * seqs))))))


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pool(g, case, layers, pages):
    """K and V of `pages` pages: [layer][page][kv head][page * head size] in the
    cache's own order, with [..][page] scales for one-byte codes."""
    _, n_kv, hd = MODELS[case["model"]]
    p, kv = {}, case["kv"]
    for n in ("k", "v"):
        shape = (layers, pages, n_kv, case["page"] * hd)
        if kv == "fp16":
            p[n] = torch.randn(shape, generator=g, device=DEV, dtype=torch.float16)
            continue
        x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float16) * (40.0 if kv == "int8" else 140.0)
        p[n] = x.round().clamp(-127, 127).to(torch.int8) if kv == "int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.int8)
        # rows of differing size
        p[n + "s"] = torch.exp(torch.randn(shape[:3] + (case["page"],), generator=g, device=DEV) * 0.3) / (40.0 if kv == "int8" else 140.0)
    return p


def _lengths(seed, n, most):
    """Ragged lengths in [1, most], the first the longest."""
    g = torch.Generator().manual_seed((int(seed) & 0x7FFFFFFF) + 1)
    return [most] + torch.randint(1, most + 1, (n - 1,), generator=g).tolist()


def _shuffled(seed, n):
    return torch.randperm(n, generator=torch.Generator().manual_seed((int(seed) & 0x7FFFFFFF) + 2)).tolist()


def _ceil(a, b):
    return -(-a // b)


def _map(rows, lens, width, pages):
    """Tables, lengths and reference counts for the sequences' page lists."""
    table = torch.full((len(rows), width), -1, dtype=torch.int32)
    ref = torch.zeros(pages, dtype=torch.int32)
    for s, r in enumerate(rows):
        if r:
            t = torch.tensor(r, dtype=torch.int32)
            table[s, :len(r)] = t
            ref.index_add_(0, t.long(), torch.ones(len(r), dtype=torch.int32))
    return {"table": table.to(DEV), "len": _ints(lens), "ref": ref.to(DEV)}


def _attn_plan(case, seed):
    """Shared pages, then each sequence's own; (rows, lengths, pages)."""
    page, full = case["page"], case["prefix"] // case["page"]
    lens = [case["prefix"] + n for n in _lengths(seed, case["batch"], case["most"])]
    more = [_ceil(n, page) - full for n in lens]
    ids, rows, at = _shuffled(seed, full + sum(more)), [], full
    for n in more:
        rows.append(ids[:full] + ids[at:at + n])
        at += n
    return rows, lens, at


def prepare(case, seed):
    kind, page = case["kind"], case["page"]
    heads, n_kv, hd = MODELS[case["model"]]
    g = _gen(seed)
    s = {"case": case}
    if kind == "attn":
        rows, lens, pages = _attn_plan(case, seed)
        s["pool"] = _pool(g, case, 1, pages)
        s["map"] = _map(rows, lens, len(rows[0]), pages)
        s["q"] = torch.randn(case["batch"], heads * hd, generator=g, device=DEV, dtype=torch.float16) * 1.5
        s["prefix"] = _ints([case["prefix"]])
        s["out"] = torch.empty_like(s["q"])
        return s
    if kind == "store":
        t, chunk = case["tokens"], case["chunk"]
        seqs = _ceil(t, chunk)
        each = _ceil(chunk + page, page)   # pages that a sequence's rows may touch
        s["pool"] = _pool(g, case, 1, seqs * each)
        ids = _shuffled(seed, seqs * each)
        start = torch.randint(0, page, (seqs,), generator=torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF)).tolist()
        slots = []
        for q in range(seqs):
            for i in range(min(chunk, t - q * chunk)):
                at = start[q] + i
                slots.append(ids[q * each + at // page] * page + at % page)
        s["slots"] = _ints(slots)
        # the rows as a fused projection leaves them: q, k and v of a token side by side
        qkv = torch.randn(t, (heads + 2 * n_kv) * hd, generator=g, device=DEV, dtype=torch.float16)
        s["qkv"] = qkv
        s["k"], s["v"] = qkv[:, heads * hd:(heads + n_kv) * hd], qkv[:, (heads + n_kv) * hd:]
        s["ko"], s["vo"] = (torch.empty(t, n_kv * hd, device=DEV, dtype=torch.float16) for _ in range(2))
        return s
    if kind == "copy":
        n = _ceil(case["tokens"], page)
        # the engine's cache of one sequence: head after head, the prompt's pages in order within each
        c = _pool(g, case, case["layers"], n + 1)
        s["cache"] = {k: x.transpose(1, 2).contiguous() for k, x in c.items()}
        s["pool"] = _pool(g, case, case["layers"], 2 * n)
        s["src"], s["dst"] = _ints(list(range(n))), _ints(_shuffled(seed, 2 * n)[:n])
        s["status"] = _ints([0])
        return s
    if kind == "branch":
        n, prompt = case["children"], case["prompt"]
        held, other = _ceil(prompt, page), 8   # other conversations' pages lie between
        pages = held + other + 2 * n + 8
        ids = _shuffled(seed, held + other + n)
        s["pool"] = _pool(g, case, case["layers"], pages)
        rows = [ids[:held], ids[held:held + other]] + [[] for _ in range(n)]
        s["map"] = _map(rows, [prompt, other * page] + [0] * n, held + other + 2, pages)
        s["parent"], s["child"] = _ints([0] * n), _ints(list(range(2, n + 2)))
        s["add"] = _ints([0, 0] + [1] * n)
        s["slots"], s["status"] = _ints([0] * n), _ints([0] * (2 * n + 4))
        return s
    n = case["seqs"]
    lens = _lengths(7, n, case["most"])   # the same for every seed, and with them the pool's size
    held = [_ceil(t, page) for t in lens]
    pages = sum(held) + 16
    ids = _shuffled(seed, sum(held))   # as traffic leaves them: interleaved
    rows, at = [], 0
    for h in held:
        rows.append(ids[at:at + h])
        at += h
    s["pool"] = _pool(g, case, case["layers"], pages)
    s["map"] = _map(rows, lens, max(held), pages)
    # even and odd sequences end in turn, and others of the same lengths come in their place
    s["ends"] = [_ints(list(range(k, n, 2))) for k in (0, 1)]
    s["adds"] = [_ints([t if q % 2 == k else 0 for q, t in enumerate(lens)]) for k in (0, 1)]
    s["tokens"] = [sum(lens[k::2]) for k in (0, 1)]
    s["slots"] = [_ints([0] * t) for t in s["tokens"]]
    s["remap"], s["status"], s["turn"] = _ints([0] * pages), _ints([0] * (n + 8)), 0
    return s


# --------------------------------------------------------------------- run
def run(state):
    return _own(state) if own else _plain(state)


def _pages(cq, s, x, layers, pages, strides=None):
    """The framework's description of a pool's tensors."""
    c = s["case"]
    _, n_kv, hd = MODELS[c["model"]]
    p = cq.kv_pages(c["page"], n_kv, hd, pages, layers, KV_TAG[c["kv"]], x["k"].data_ptr(), x["v"].data_ptr(),
                    x["ks"].data_ptr() if "ks" in x else None, x["vs"].data_ptr() if "vs" in x else None)
    if strides:
        p.layer_stride, p.page_stride, p.head_stride = strides
    return p


def _handles(cq, s):
    """What a program makes once for a cache: its descriptions and the workspaces."""
    c, kind = s["case"], s["case"]["kind"]
    heads, n_kv, hd = MODELS[c["model"]]
    x = s["pool"]
    h = {"pages": _pages(cq, s, x, x["k"].shape[0], x["k"].shape[1])}
    if kind == "copy":
        run = s["cache"]["k"].shape[2] * c["page"] * hd   # elements of one head
        h["cache"] = _pages(cq, s, s["cache"], c["layers"], s["cache"]["k"].shape[2], (n_kv * run, c["page"] * hd, run))
    if "map" in s:
        m = s["map"]
        h["map"] = cq.page_map(m["ref"].data_ptr(), m["table"].data_ptr(), m["len"].data_ptr(), x["k"].shape[1], m["table"].shape[0],
                               m["table"].shape[1], c["page"])
    n = 0
    if kind == "attn":
        n = cq.lib.cq_prefix_attention_workspace_bytes(c["batch"], heads, n_kv, hd)
    elif kind in ("branch", "compact"):
        n = cq.lib.cq_pages_workspace_bytes(ctypes.byref(h["map"]))
    h["work"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    return {k: ctypes.byref(v) if isinstance(v, ctypes.Structure) else v for k, v in h.items()}


def _own(s):
    import cuqwen_amd as cq
    c, kind, lib, ck = s["case"], s["case"]["kind"], cq.lib, cq.check
    heads, n_kv, hd = MODELS[c["model"]]
    if "handles" not in s:
        s["handles"] = _handles(cq, s)
    h = s["handles"]
    if kind == "attn":
        m = s["map"]
        ck(lib.cq_prefix_attention_decode(
            s["q"].data_ptr(), heads * hd, s["out"].data_ptr(), heads * hd, h["pages"], m["table"].data_ptr(), m["table"].shape[1],
            s["prefix"].data_ptr(), h["pages"], m["table"].data_ptr(), m["table"].shape[1], s["prefix"].data_ptr(), m["len"].data_ptr(),
            c["batch"], 0, heads, h["work"].data_ptr(), None))
        return s["out"]
    if kind == "store":
        row = s["k"].stride(0)
        ck(lib.cq_paged_kv_store(h["pages"], 0, s["k"].data_ptr(), s["v"].data_ptr(), row, s["slots"].data_ptr(), c["tokens"], None))
        if c["kv"] == "fp16":
            return {"k": s["pool"]["k"], "v": s["pool"]["v"]}
        ck(lib.cq_paged_kv_load(h["pages"], 0, s["ko"].data_ptr(), s["vo"].data_ptr(), n_kv * hd, s["slots"].data_ptr(), c["tokens"], None))
        return {"k": s["ko"], "v": s["vo"], "ks": s["pool"]["ks"], "vs": s["pool"]["vs"]}
    if kind == "copy":
        ck(lib.cq_pages_copy(h["cache"], h["pages"], s["src"].data_ptr(), s["dst"].data_ptr(), s["src"].numel(), s["status"].data_ptr(), None))
        return dict(_whole(s["pool"], c), status=s["status"])
    st = s["status"].data_ptr()
    if kind == "branch":
        n = c["children"]
        ck(lib.cq_pages_trim(h["map"], s["child"].data_ptr(), None, n, st, None))
        ck(lib.cq_pages_fork(h["map"], s["parent"].data_ptr(), s["child"].data_ptr(), n, st + 4 * n, None))
        ck(lib.cq_pages_append(h["pages"], h["map"], s["add"].data_ptr(), s["slots"].data_ptr(), n, st + 8 * n, h["work"].data_ptr(), None))
        return dict(_whole(s["pool"], c), **s["map"], slots=s["slots"], status=s["status"])
    k = s["turn"] = 1 - s["turn"]
    n = s["ends"][k].numel()
    ck(lib.cq_pages_trim(h["map"], s["ends"][k].data_ptr(), None, n, st, None))
    ck(lib.cq_pages_compact(h["pages"], h["map"], s["remap"].data_ptr(), st + 4 * n, h["work"].data_ptr(), None))
    ck(lib.cq_pages_append(h["pages"], h["map"], s["adds"][k].data_ptr(), s["slots"][k].data_ptr(), s["tokens"][k], st + 4 * n + 16,
                           h["work"].data_ptr(), None))
    return dict(_whole(s["pool"], c), **s["map"], remap=s["remap"], slots=s["slots"][k], status=s["status"][:n + 8])


def _whole(pool, case):
    """A pool's tensors, E4M3 codes as the numbers that they are."""
    return {n: x.view(torch.float8_e4m3fn) if case["kv"] == "fp8" and n in ("k", "v") else x for n, x in pool.items()}


# -------------------------------------------------------------- plain form
def _untile(x, kind, kv, page, hd):
    """[..., page * hd] in the cache's order -> [..., page, hd], 32 bits."""
    lead, n = x.shape[:-1], x.dim() - 1
    at = lambda *p: list(range(n)) + [n + i for i in p]   # noqa: E731
    if kv == "fp8":
        x = x.view(torch.float8_e4m3fn)
    x = x.float()
    if kind == "k" and kv == "fp16":       # 16-token tiles [kk][j][token][8]
        x = x.view(*lead, page // 16, hd // 32, 4, 16, 8).permute(at(0, 3, 1, 2, 4))
    elif kind == "k":                      # [kk / 2][j][token][kk % 2][8]
        x = x.view(*lead, page // 16, hd // 64, 4, 16, 2, 8).permute(at(0, 3, 1, 4, 2, 5))
    elif kv == "fp16":                     # 32-token tiles [dt][j][dl][hi][lo], token = hi * 16 + j * 4 + lo
        x = x.view(*lead, page // 32, hd // 16, 4, 16, 2, 4).permute(at(0, 4, 2, 5, 1, 3))
    else:                                  # [dt / 2][j][dl][dt % 2][hi][lo]
        x = x.view(*lead, page // 32, hd // 32, 4, 16, 2, 2, 4).permute(at(0, 5, 2, 6, 1, 4, 3))
    return x.reshape(*lead, page, hd)


def _rows(pool, name, case, ids):
    """The rows of pages ids[...] of layer 0: [..., kv head, page, head size], 32 bits."""
    hd = MODELS[case["model"]][2]
    x = _untile(pool[name][0][ids], name, case["kv"], case["page"], hd)
    return x if case["kv"] == "fp16" else x * pool[name + "s"][0][ids].unsqueeze(-1)


def _plain_attn(s):
    c, m, pool = s["case"], s["map"], s["pool"]
    heads, n_kv, hd = MODELS[c["model"]]
    b, g, page, lp = c["batch"], heads // n_kv, c["page"], c["prefix"]
    table, first = m["table"].long(), lp // page
    q = (s["q"].float() / math.sqrt(hd)).view(b, n_kv, g, hd)
    shared = table[0, :_ceil(lp, page)]
    kp, vp = (_rows(pool, n, c, shared).transpose(0, 1).reshape(n_kv, -1, hd)[:, :lp] for n in ("k", "v"))
    mine = table[:, first:].clamp(min=0)
    ko, vo = (_rows(pool, n, c, mine).transpose(1, 2).reshape(b, n_kv, -1, hd) for n in ("k", "v"))
    at = first * page + torch.arange(ko.shape[2], device=DEV)
    seen = (at >= s["prefix"]) & (at < m["len"].unsqueeze(1))
    sp = torch.matmul(q.transpose(0, 1).reshape(n_kv, b * g, hd), kp.transpose(1, 2).contiguous())
    so = torch.matmul(q, ko.transpose(2, 3).contiguous()).masked_fill(~seen[:, None, None, :], -math.inf)
    top = torch.maximum(sp.amax(-1).view(n_kv, b, g).transpose(0, 1), so.amax(-1))
    pp = torch.exp(sp - top.transpose(0, 1).reshape(n_kv, b * g, 1))
    po = torch.exp(so - top.unsqueeze(-1))
    total = pp.sum(-1).view(n_kv, b, g).transpose(0, 1) + po.sum(-1)
    out = torch.matmul(pp, vp).view(n_kv, b, g, hd).transpose(0, 1) + torch.matmul(po, vo)
    return (out / total.unsqueeze(-1)).reshape(b, heads * hd).half()


def _places(slots, kind, kv, page, hd):
    """Element offsets within a head's page of rows slots % page: [token, hd]."""
    t = (slots.long() % page).unsqueeze(1)
    d = torch.arange(hd, device=DEV)
    if kind == "k":
        kk, j, e = d // 32, d // 8 % 4, d % 8
        piece, tile = kk, t // 16 * (16 * hd)
        lane = j * 16 + t % 16
    else:
        piece, e = d // 16, t % 4 + t % 32 // 16 * 4
        lane, tile = t % 16 // 4 * 16 + d % 16, t // 32 * (32 * hd)
    if kv == "fp16":
        return tile + (piece * 64 + lane) * 8 + e
    return tile + (piece // 2 * 64 + lane) * 16 + piece % 2 * 8 + e


def _plain_store(s):
    c, pool = s["case"], s["pool"]
    _, n_kv, hd = MODELS[c["model"]]
    kv, page, out = c["kv"], c["page"], {}
    slots = s["slots"].long()
    for n in ("k", "v"):
        x = s[n].reshape(-1, n_kv, hd)
        at = ((slots // page).view(-1, 1, 1) * n_kv + torch.arange(n_kv, device=DEV).view(1, -1, 1)) * (page * hd) + \
            _places(s["slots"], n, kv, page, hd).unsqueeze(1)
        flat = pool[n].view(-1)
        if kv == "fp16":
            flat[at.view(-1)] = x.reshape(-1)
            out[n] = pool[n]
            continue
        top = torch.full((), 127.0 if kv == "int8" else 448.0, device=DEV)
        scale = x.float().abs().amax(-1) / top
        y = x.float() / torch.where(scale > 0, scale, torch.ones_like(scale)).unsqueeze(-1)
        code = y.round().clamp(-127, 127).to(torch.int8) if kv == "int8" else y.to(torch.float8_e4m3fn).view(torch.int8)
        flat[at.view(-1)] = code.view(-1)
        row = ((slots // page).view(-1, 1) * n_kv + torch.arange(n_kv, device=DEV)) * page + (slots % page).view(-1, 1)
        pool[n + "s"].view(-1)[row.view(-1)] = scale.view(-1)
        back = flat[at.view(-1)].view(at.shape)
        back = back.float() if kv == "int8" else back.view(torch.float8_e4m3fn).float()
        out[n] = (back * pool[n + "s"].view(-1)[row.view(-1)].view(-1, n_kv, 1)).reshape(-1, n_kv * hd).half()
        out[n + "s"] = pool[n + "s"]
    return out


def _plain_trim(m, seqs):
    at = seqs.long()
    rows = m["table"][at]
    held = torch.arange(rows.shape[1], device=DEV) < ((m["len"][at] + m["page"] - 1) // m["page"]).unsqueeze(1)
    m["ref"].index_add_(0, rows.clamp(min=0).view(-1), -held.int().view(-1))
    m["table"][at] = torch.where(held, -torch.ones_like(rows), rows)
    m["len"][at] = 0
    return torch.zeros_like(seqs)


def _plain_fork(m, parents, children):
    rows, n = m["table"][parents.long()], m["len"][parents.long()]
    held = torch.arange(rows.shape[1], device=DEV) < ((n + m["page"] - 1) // m["page"]).unsqueeze(1)
    m["ref"].index_add_(0, rows.clamp(min=0).view(-1), held.int().view(-1))
    at = children.long()
    m["table"][at] = torch.where(held, rows, m["table"][at])
    m["len"][at] = n
    return torch.zeros_like(parents)


def _plain_append(pool, m, add, n_slots):
    table, length, ref, page = m["table"], m["len"], m["ref"], m["page"]
    n, width = table.shape
    cols, seqs = torch.arange(width, device=DEV), torch.arange(n, device=DEV)
    before, after = (length + page - 1) // page, (length + add + page - 1) // page
    last = table[seqs, (before - 1).clamp(min=0).long()].clamp(min=0)
    writes = (add > 0) & (length % page > 0)
    earlier = (last.unsqueeze(0) == last.unsqueeze(1)) & writes.unsqueeze(0) & (seqs.unsqueeze(0) < seqs.unsqueeze(1))
    copies = writes & (ref[last.long()] - earlier.sum(1) > 1)
    wants = ((cols >= before.unsqueeze(1)) & (cols < after.unsqueeze(1))) | (copies.unsqueeze(1) & (cols == before.unsqueeze(1) - 1))
    rank = (torch.cumsum(wants.view(-1).int(), 0) - 1).clamp(min=0).view(n, width)
    free = torch.sort((ref > 0).int(), stable=True).indices
    fresh = free[rank.clamp(max=free.numel() - 1)].int()
    taken = wants.sum()
    ref.index_add_(0, last, -copies.int())
    ref.index_add_(0, torch.where(wants, fresh, torch.zeros_like(fresh)).view(-1), wants.int().view(-1))
    table.copy_(torch.where(wants, fresh, table))
    # the filled tiles of the pages that become their writer's own
    who = torch.nonzero(copies).view(-1)
    src, dst = last[who].long(), table[who, before[who].long() - 1].long()
    part = (torch.arange(page // 32, device=DEV) < ((length[who] % page + 31) // 32).unsqueeze(1)).view(1, -1, 1, page // 32, 1)
    for x in pool.values():
        y = x.view(x.shape[0], x.shape[1], x.shape[2], page // 32, -1)
        y[:, dst] = torch.where(part, y[:, src], y[:, dst])
    ends = torch.cumsum(add, 0)
    t = torch.arange(n_slots, device=DEV)
    q = torch.searchsorted(ends, t, right=True).clamp(max=n - 1)
    pos = length[q] + t - (ends - add)[q]
    slots = torch.where(t < ends[-1], table[q, (pos // page).clamp(max=width - 1)] * page + pos % page, -torch.ones_like(pos)).int()
    length += add
    return slots, torch.stack([torch.zeros_like(taken), taken, copies.sum(), ends[-1].long()]).int()


def _plain_compact(pool, m):
    ref, page = m["ref"], m["page"]
    used = ref > 0
    count = used.sum()
    at = torch.arange(ref.numel(), device=DEV)
    to, frm = torch.nonzero(~used & (at < count)).view(-1), torch.nonzero(used & (at >= count)).view(-1)
    remap = torch.where(used, at, -torch.ones_like(at)).int()
    remap[frm] = to.int()
    held = torch.arange(m["table"].shape[1], device=DEV) < ((m["len"] + page - 1) // page).unsqueeze(1)
    m["table"].copy_(torch.where(held, remap[m["table"].clamp(min=0).long()], m["table"]))
    ref[to] = ref[frm]
    ref[frm] = 0
    for x in pool.values():
        x[:, to] = x[:, frm]
    return remap, torch.stack([count * 0, count, count * 0 + to.numel(), count * 0]).int()


def _plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "attn":
        return _plain_attn(s)
    if kind == "store":
        return _plain_store(s)
    if kind == "copy":
        src, dst = s["src"].long(), s["dst"].long()
        for n, x in s["pool"].items():
            y = s["cache"][n]
            x[:, dst] = y.transpose(1, 2)[:, src]
        return dict(_whole(s["pool"], c), status=torch.zeros_like(s["status"]))
    m = dict(s["map"], page=c["page"])
    if kind == "branch":
        a = _plain_trim(m, s["child"])
        b = _plain_fork(m, s["parent"], s["child"])
        slots, d = _plain_append(s["pool"], m, s["add"], c["children"])
        return dict(_whole(s["pool"], c), **s["map"], slots=slots, status=torch.cat([a, b, d]))
    k = s["turn"] = 1 - s["turn"]
    a = _plain_trim(m, s["ends"][k])
    remap, b = _plain_compact(s["pool"], m)
    slots, d = _plain_append(s["pool"], m, s["adds"][k], s["tokens"][k])
    return dict(_whole(s["pool"], c), **s["map"], remap=remap, slots=slots, status=torch.cat([a, b, d]))


# -------------------------------------------------------------------- work
def work(case):
    heads, n_kv, hd = MODELS[case["model"]]
    kind, page = case["kind"], case["page"]
    row = 2 * n_kv * (2 * hd if case["kv"] == "fp16" else hd + 4)   # bytes of a token's K and V
    if kind == "attn":
        mine = case["batch"] * (case["most"] + 1) / 2
        return {"bytes": (case["prefix"] + mine) * row + 4 * case["batch"] * heads * hd,
                "flops": 4.0 * heads * hd * (case["batch"] * case["prefix"] + mine)}
    if kind == "store":
        t = case["tokens"]
        back = 0 if case["kv"] == "fp16" else 4 * n_kv * hd + row
        return {"bytes": t * (4 * n_kv * hd + row + 4 + back), "flops": 0 if case["kv"] == "fp16" else 6.0 * t * n_kv * hd}
    if kind == "copy":
        return {"bytes": 2 * _ceil(case["tokens"], page) * page * row * case["layers"], "flops": 0}
    if kind == "branch":
        n, held = case["children"], _ceil(case["prompt"], page)
        tail = _ceil(case["prompt"] % page, 32) * 32
        return {"bytes": 2 * n * tail * row * case["layers"] + n * held * 4 * 4, "flops": 0}
    half = case["seqs"] / 2 * (case["most"] + page) / 2   # tokens in the pages that move
    return {"bytes": 2 * half * row * case["layers"] + 8 * case["seqs"] * case["most"] / page * 4, "flops": 0}


# ------------------------------------------------- the definition, 64 bits
def _value_at(pool, name, case, page_id, head):
    """Rows of one head's page in 64 bits, element by element of its order."""
    hd, page, kv = MODELS[case["model"]][2], case["page"], case["kv"]
    x = pool[name][0, page_id, head]
    if kv == "fp8":
        x = x.view(torch.float8_e4m3fn).double()
    at = _places(torch.arange(page, device=DEV), name, kv, page, hd)
    x = x.double()[..., at]
    return x if kv == "fp16" else x * pool[name + "s"][0, page_id, head].double().unsqueeze(-1)


def _exact_attn(case, seed):
    s = prepare(case, seed)
    heads, n_kv, hd = MODELS[case["model"]]
    rows, lens, _ = _attn_plan(case, seed)
    g, page, lp = heads // n_kv, case["page"], case["prefix"]
    out = torch.zeros(case["batch"], heads, hd, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(case["batch"], heads, hd)
    for h in range(n_kv):
        shared = torch.tensor(rows[0][:_ceil(lp, page)], device=DEV)
        kp, vp = (_value_at(s["pool"], n, case, shared, h).reshape(-1, hd)[:lp] for n in ("k", "v"))
        for b in range(case["batch"]):
            mine = torch.tensor(rows[b][lp // page:], device=DEV)
            ko, vo = (_value_at(s["pool"], n, case, mine, h).reshape(-1, hd)[lp % page:lens[b] - lp // page * page] for n in ("k", "v"))
            w = torch.softmax(q[b, h * g:(h + 1) * g] @ torch.cat([kp, ko]).T / math.sqrt(hd), -1)
            out[b, h * g:(h + 1) * g] = w[:, :lp] @ vp + w[:, lp:] @ vo
    return out.view(case["batch"], heads * hd)


class _Book:
    """The page map kept by hand."""

    def __init__(self, m, page):
        self.rows = [[p for p in r if p >= 0] for r in m["table"].tolist()]
        self.len, self.ref, self.page, self.width = m["len"].tolist(), m["ref"].tolist(), page, m["table"].shape[1]

    def trim(self, s):
        for p in self.rows[s]:
            self.ref[p] -= 1
        self.rows[s], self.len[s] = [], 0

    def fork(self, parent, child):
        self.rows[child], self.len[child] = list(self.rows[parent]), self.len[parent]
        for p in self.rows[child]:
            self.ref[p] += 1

    def append(self, add):
        free = iter([p for p, r in enumerate(self.ref) if r == 0])
        moved, slots, taken = [], [], 0
        for s, n in enumerate(add):
            for i in range(n):
                at = self.len[s]
                if at % self.page == 0:
                    self.rows[s].append(next(free))
                    self.ref[self.rows[s][-1]], taken = 1, taken + 1
                elif i == 0 and self.ref[self.rows[s][-1]] > 1:
                    old, new = self.rows[s][-1], next(free)
                    self.ref[old], self.ref[new], self.rows[s][-1], taken = self.ref[old] - 1, 1, new, taken + 1
                    moved.append((old, new, _ceil(at % self.page, 32)))
                slots.append(self.rows[s][at // self.page] * self.page + at % self.page)
                self.len[s] += 1
        return moved, slots, [0, taken, len(moved), sum(add)]

    def compact(self):
        count = sum(r > 0 for r in self.ref)
        to = [p for p in range(count) if self.ref[p] == 0]
        frm = [p for p in range(count, len(self.ref)) if self.ref[p] > 0]
        remap = [p if r > 0 else -1 for p, r in enumerate(self.ref)]
        for a, b in zip(frm, to):
            remap[a], self.ref[b], self.ref[a] = b, self.ref[a], 0
        self.rows = [[remap[p] for p in r] for r in self.rows]
        return list(zip(frm, to)), remap, [0, count, len(to), 0]

    def as_tensors(self):
        return {"table": _ints([r + [-1] * (self.width - len(r)) for r in self.rows]), "len": _ints(self.len), "ref": _ints(self.ref)}


def exact(case, seed):
    kind, page = case["kind"], case["page"]
    if kind == "attn":
        return _exact_attn(case, seed)
    s = prepare(case, seed)
    if kind == "store":
        _, n_kv, hd = MODELS[case["model"]]
        out = {}
        for n in ("k", "v"):
            x = s[n].double().reshape(-1, n_kv, hd)
            if case["kv"] == "fp16":
                pool = s["pool"][n].clone()
                at = _places(s["slots"], n, "fp16", page, hd)
                for h in range(n_kv):
                    pool[0, (s["slots"].long() // page).unsqueeze(1), h, at] = x[:, h].half()
                out[n] = pool
                continue
            # the values that the codes stand for, within a step of the row itself; the codes' own rounding is not a computed number
            scale = x.abs().amax(-1) / (127.0 if case["kv"] == "int8" else 448.0)
            y = x / scale.clamp(min=1e-300).unsqueeze(-1)
            if case["kv"] == "int8":
                y = y.round().clamp(-127, 127)
            else:
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                y = (y / step).round() * step
            out[n] = (y * scale.unsqueeze(-1)).reshape(-1, n_kv * hd)
            pool = s["pool"][n + "s"].double()
            at = s["slots"].long()
            pool[0, at // page, :, at % page] = scale
            out[n + "s"] = pool
        return out
    pool = {n: x.clone() for n, x in s["pool"].items()}
    if kind == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            for n, x in pool.items():
                x[:, b] = s["cache"][n][:, :, a]
        return dict(_whole(pool, case), status=None)
    book = _Book(s["map"], page)
    if kind == "branch":
        n = case["children"]
        for a, b in zip(s["parent"].tolist(), s["child"].tolist()):
            book.trim(b)
            book.fork(a, b)
        moved, slots, said = book.append(s["add"].tolist())
        extra, status = {}, [0] * (2 * n) + said
    else:
        for q in s["ends"][1].tolist():
            book.trim(q)
        pairs, remap, first = book.compact()
        for a, b in pairs:
            for x in pool.values():
                x[:, b] = x[:, a].clone()
        moved, slots, said = book.append(s["adds"][1].tolist())
        extra, status = {"remap": _ints(remap)}, [0] * s["ends"][1].numel() + first + said
    for a, b, tiles in moved:
        for x in pool.values():
            y = x.view(x.shape[0], x.shape[1], x.shape[2], page // 32, -1)
            y[:, b, :, :tiles] = y[:, a, :, :tiles]
    return dict(_whole(pool, case), **book.as_tensors(), **extra, slots=_ints(slots), status=_ints(status))
