"""Operators of a server that keeps many sequences in one paged key/value cache, as its decode step runs them one after the other:

  append     new rows of queries, keys and values: rms norm of each query and key head (or none), rotation by position, queries back to the
             caller, keys and values into the sequences' pages                                        (l2b_paged_append_device)
  attention  of those queries over the pages of a prefix that all sequences share and over each sequence's own pages   (l2b_paged_attention_device)
  sample     the next token of every sequence: temperature, top-k, top-p, min-p, a given random number                 (l2b_sample_device)

A case is a dict of plain values; sizes are those of this library's models (8 to 64 heads of 64, 96 or 128 values, vocabularies of 32 000 and
128 256) or lie between them.  `run` computes the plain form, elementary torch operations in 32 or 64 bits, or, where `own` is set, makes the
library's calls.  Pages are handed out in random order; a page table holds -1 behind a sequence's last page."""
import ctypes as C
import importlib.util
import math
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
own = False
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GGML = {"f32": 0, "f16": 1, "bf16": 30}  # l2b_ggml_type
EPS = 1e-6


def listed():
    return [
        # one chat, one new token: latency
        _append("append_chat", n_seq=1, n_query=1, heads=32, kv_heads=8, size=128, prefix=0, past=500, io="bf16", cache="bf16", neox=False, norm=False, page=16),
        # a server's slots, one new token each; activations are f32 as everywhere in this library
        _append("append_slots_f32", n_seq=48, n_query=1, heads=16, kv_heads=4, size=128, prefix=777, past=900, io="f32", cache="bf16", neox=False, norm=True, page=32),
        # prompts of several users, padded to the longest
        _append("append_prompts", n_seq=5, n_query=701, heads=24, kv_heads=24, size=96, prefix=0, past=0, io="f16", cache="f16", neox=True, norm=True, page=64),
        # one long document
        _append("append_document", n_seq=1, n_query=12000, heads=64, kv_heads=8, size=128, prefix=0, past=0, io="bf16", cache="bf16", neox=True, norm=True, page=64),
        # one chat
        _attention("attend_chat", n_seq=1, n_query=1, heads=32, kv_heads=8, size=128, prefix=0, past=500, io="bf16", cache="bf16", page=16),
        # slots with chats of all lengths that share nothing
        _attention("attend_slots", n_seq=24, n_query=1, heads=24, kv_heads=24, size=96, prefix=0, past=4000, io="f16", cache="f16", page=64),
        # short questions about one document
        _attention("attend_document", n_seq=64, n_query=1, heads=32, kv_heads=8, size=128, prefix=6001, past=400, io="bf16", cache="bf16", page=64),
        # drafts of four tokens checked at once behind a system prompt; f32 queries over a bf16 cache, as in the layer-stack models
        _attention("attend_drafts_f32", n_seq=32, n_query=4, heads=64, kv_heads=8, size=128, prefix=1111, past=1500, io="f32", cache="bf16", page=32),
        # many samples of one long context: nearly all work is in the shared part
        _attention("attend_samples", n_seq=128, n_query=1, heads=64, kv_heads=8, size=128, prefix=16000, past=200, io="bf16", cache="bf16", page=128),
        # one chat, the filters that chats use
        _sample("sample_chat", rows=1, vocab=128256, io="f32", top_k=40, top_p=0.95, min_p=0.0, greedy=False),
        # a batch in which every row has settings of its own, some of them greedy
        _sample("sample_slots", rows=64, vocab=128256, io="f32", top_k=100, top_p=0.9, min_p=0.02, greedy=True),
        # many samples of a smaller vocabulary, by temperature and nucleus alone
        _sample("sample_many", rows=200, vocab=32000, io="bf16", top_k=0, top_p=0.98, min_p=0.0, greedy=False),
    ]


def _append(name, **k):
    return dict(name=name, kind="append", **k)


def _attention(name, **k):
    return dict(name=name, kind="attention", **k)


def _sample(name, **k):
    return dict(name=name, kind="sample", **k)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "sample"])
    if kind == "sample":
        vocab = _log(rng, 300, 128256)
        return dict(kind=kind, rows=_log(rng, 1, min(256, max(1, 8208384 // vocab))), vocab=vocab, io=rng.choice(["f32", "f32", "bf16", "f16"]), top_k=rng.choice([0, 1, 20, 50, _log(rng, 1, 4000)]),
                    top_p=rng.choice([1.0, 0.5, 0.9, rng.uniform(0.1, 0.999)]), min_p=rng.choice([0.0, 0.0, 0.05, rng.uniform(0.001, 0.3)]), greedy=rng.random() < 0.3)
    heads, kv_heads = rng.choice([(32, 8), (24, 24), (16, 4), (64, 8), (8, 8), (6, 6), (12, 2)])
    cache = rng.choice(["bf16", "bf16", "f16"])
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, size=rng.choice([128, 128, 96, 64, 48, 80]), io=rng.choice([cache, cache, "f32"]), cache=cache, page=rng.choice([8, 16, 32, 64, 128, 256]))
    if kind == "append":
        n_seq = _log(rng, 1, 256)
        return dict(c, n_seq=n_seq, n_query=_log(rng, 1, max(1, 6000 // n_seq)), prefix=rng.choice([0, _log(rng, 1, 20000)]), past=rng.choice([0, _log(rng, 1, 1000)]), neox=rng.random() < 0.5, norm=rng.random() < 0.5)
    n_seq = _log(rng, 1, 128)
    n_query = rng.choice([1, 1, 1, 2, 3, 5])
    keys = 8 * 16000 // kv_heads  # of the largest listed case, in positions
    return dict(c, n_seq=n_seq, n_query=n_query, prefix=rng.choice([0, _log(rng, 1, min(16000, max(1, 128 * 64 * keys // (n_seq * n_query * heads * 8))))]), past=_log(rng, 1, max(1, min(8000, keys // n_seq))))


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) & 0xFFFFFFFF) * 1000003 + what)
    return g


def _normal(shape, g, t, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)


def _lengths(c, seed):
    """Own positions of each sequence before the new rows, and its number of new rows: whole numbers on the host, as a scheduler has them."""
    r = np.random.RandomState((int(seed) * 7919 + 13) & 0x7FFFFFFF)
    n = c["n_seq"]
    past = np.full(n, c["past"]) if n == 1 else r.randint(c["past"] // 8, c["past"] + 1, n)
    if c["n_query"] == 1:
        counts = np.ones(n, np.int64)
    else:
        counts = r.randint((c["n_query"] + 1) // 2, c["n_query"] + 1, n)
        counts[r.randint(n)] = c["n_query"]
    return past.astype(np.int64), counts.astype(np.int64)


def _paged(c, seed):
    """The cache's pages (one more than the library is told of, where the plain form's rows without a place go), page tables and lengths."""
    past, counts = _lengths(c, seed)
    page, lengths = c["page"], past + counts
    prefix_pages, each = -(-c["prefix"] // page), -(-lengths // page)
    width = -(-(c["past"] + c["n_query"]) // page)  # pages of the longest sequence there may be
    n_pages = prefix_pages + c["n_seq"] * width + 2
    r = np.random.RandomState((int(seed) * 104729 + 5) & 0x7FFFFFFF)
    order = r.permutation(n_pages)
    table = np.full((c["n_seq"], width), -1, np.int32)
    table[np.arange(width) < each[:, None]] = order[prefix_pages:prefix_pages + each.sum()]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    shape = (n_pages + 1, c["kv_heads"], page, c["size"])
    g = _gen(seed, 1)
    return dict(case=c, n_pages=n_pages, k=_normal(shape, g, TYPES[c["cache"]]), v=_normal(shape, g, TYPES[c["cache"]]), table=dev(table), lengths=dev(lengths), counts=dev(counts),
                prefix_pages=dev(order[:prefix_pages]))


def prepare(case, seed):
    c = case
    if c["kind"] == "sample":
        rows, g = c["rows"], _gen(seed, 2)
        logits = torch.randn((rows, c["vocab"]), generator=g, device="cuda") * 2.5
        few = torch.randint(0, c["vocab"], (rows, min(40, c["vocab"])), generator=g, device="cuda")  # the words that fit the context
        logits.scatter_add_(1, few, torch.rand(few.shape, generator=g, device="cuda") * 9)
        rand = lambda: torch.rand(rows, generator=g, device="cuda")  # noqa: E731
        temperature = 0.6 + 0.6 * rand()
        if c["greedy"]:
            temperature = torch.where(rand() < 0.2, torch.zeros_like(temperature), temperature)
        # rows of a batch have settings of their own, around the case's
        top_k = torch.full((rows,), c["top_k"], device="cuda") if rows == 1 else (c["top_k"] * (0.5 + rand())).round()
        top_p = torch.full((rows,), c["top_p"], device="cuda") if rows == 1 or c["top_p"] >= 1 else c["top_p"] + (1 - c["top_p"]) * rand() * 0.5
        min_p = torch.full((rows,), c["min_p"], device="cuda") * (0.5 + rand())
        s = dict(case=c, logits=logits.to(TYPES[c["io"]]), temperature=temperature, top_k=top_k.to(torch.int32), top_p=top_p, min_p=min_p,
                 uniform=torch.rand(rows, generator=g, device="cuda", dtype=torch.float64), tokens=torch.zeros(rows, dtype=torch.int32, device="cuda"), probs=torch.zeros(rows, device="cuda"))
    else:
        s = _paged(c, seed)
        g, rows, t = _gen(seed, 3), c["n_seq"] * c["n_query"], TYPES[c["io"]]
        if c["kind"] == "append":
            width = (c["heads"] + 2 * c["kv_heads"]) * c["size"]
            qkv = _normal((rows, width), g, t)  # one product's result: queries, keys and values of a row side by side
            at = np.cumsum([0, c["heads"], c["kv_heads"], c["kv_heads"]]) * c["size"]
            s.update(q=qkv[:, at[0]:at[1]], new_k=qkv[:, at[1]:at[2]], new_v=qkv[:, at[2]:at[3]], q_out=torch.zeros((rows, c["heads"] * c["size"]), dtype=t, device="cuda"))
            s.update(gains=[1 + 0.1 * torch.randn(c["size"], generator=g, device="cuda") for _ in range(2)] if c["norm"] else [None, None])
        else:
            s.update(q=_normal((rows, c["heads"] * c["size"]), g, t, 2.0), out=torch.zeros((rows, c["heads"] * c["size"]), dtype=t, device="cuda"))
    if own:  # the descriptors and the workspace, which a decode loop keeps beside its buffers
        s["plan"] = _plan(s)
    return s


# ---- the library's calls ------------------------------------------------------------------------------------------------------
def _library():
    name = "llama2_jl_b200"  # the package's folder has a dot in its name
    if name not in sys.modules:
        d = os.path.join(ROOT, "llama2.jl_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(d, "__init__.py"), submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]._lib


def _plan(s):
    L, c = _library(), s["case"]
    at = lambda t: None if t is None or t.numel() == 0 else t.data_ptr()  # noqa: E731
    if c["kind"] == "sample":
        return [L.Sampling(type=GGML[c["io"]], n_rows=c["rows"], vocab=c["vocab"], dev_logits=at(s["logits"]), stride=c["vocab"], dev_temperature=at(s["temperature"]), dev_top_k=at(s["top_k"]),
                           dev_top_p=at(s["top_p"]), dev_min_p=at(s["min_p"]), dev_uniform=at(s["uniform"]), dev_tokens=at(s["tokens"]), dev_probs=at(s["probs"]))]
    cache = L.PagedCache(dev_k=at(s["k"]), dev_v=at(s["v"]), type=GGML[c["cache"]], n_pages=s["n_pages"], page_size=c["page"], n_kv_heads=c["kv_heads"], head_size=c["size"])
    batch = L.PagedBatch(n_seq=c["n_seq"], n_query=c["n_query"], dev_lengths=at(s["lengths"]), dev_counts=at(s["counts"]), dev_pages=at(s["table"]), pages_per_seq=s["table"].shape[1],
                         prefix_len=c["prefix"], dev_prefix_pages=at(s["prefix_pages"]))
    if c["kind"] == "append":
        rows = L.PagedRows(type=GGML[c["io"]], n_heads=c["heads"], dev_q=at(s["q"]), dev_k=at(s["new_k"]), dev_v=at(s["new_v"]), q_stride=s["q"].stride(0), k_stride=s["new_k"].stride(0),
                           v_stride=s["new_v"].stride(0), dev_q_out=at(s["q_out"]), q_out_stride=s["q_out"].stride(0), dev_q_gain=at(s["gains"][0]), dev_k_gain=at(s["gains"][1]), eps=EPS,
                           rope_freq_base=10000.0, rope_is_neox=int(c["neox"]))
        return [cache, batch, rows]
    queries = L.PagedQueries(type=GGML[c["io"]], n_heads=c["heads"], dev_q=at(s["q"]), q_stride=s["q"].stride(0), dev_out=at(s["out"]), out_stride=s["out"].stride(0), scale=0.0)
    need = C.c_int64()
    L.check(L.lib().l2b_paged_attention_workspace(C.byref(cache), C.byref(batch), C.byref(queries), C.byref(need)))
    s["workspace"] = torch.empty(max(16, need.value), dtype=torch.uint8, device="cuda")
    return [cache, batch, queries]


def _call(s):
    L, kind, p = _library(), s["case"]["kind"], s["plan"]
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "append":
        L.check(L.lib().l2b_paged_append_device(C.byref(p[0]), C.byref(p[1]), C.byref(p[2]), stream))
    elif kind == "attention":
        w = s["workspace"]
        L.check(L.lib().l2b_paged_attention_device(C.byref(p[0]), C.byref(p[1]), C.byref(p[2]), w.data_ptr(), w.numel(), stream))
    else:
        L.check(L.lib().l2b_sample_device(C.byref(p[0]), stream))


def run(state):
    s = state
    if own:
        _call(s)
    else:
        {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[s["case"]["kind"]](s)
    if s["case"]["kind"] == "append":
        return {"q": s["q_out"], "k": s["k"][:s["n_pages"]], "v": s["v"][:s["n_pages"]]}
    return {"out": s["out"]} if s["case"]["kind"] == "attention" else {"tokens": s["tokens"], "probs": s["probs"]}


# ---- plain forms --------------------------------------------------------------------------------------------------------------
def _places(s):
    """Own position of every row [n_seq, n_query], and whether the row is a new token."""
    j = torch.arange(s["case"]["n_query"], device="cuda")
    return (s["lengths"] - s["counts"])[:, None].long() + j, j < s["counts"][:, None]


def _turned(x, gain, cos, sin, neox):
    """x [rows, heads, size] in f32: normed (where there is a gain) and rotated."""
    if gain is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if neox else (x[..., 0::2], x[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.cat((a, b), -1) if neox else torch.stack((a, b), -1).flatten(-2)


def _plain_append(s):
    c = s["case"]
    pos, new = _places(s)
    size, page, rows = c["size"], c["page"], pos.numel()
    freq = 10000.0 ** (-torch.arange(0, size, 2, device="cuda", dtype=torch.float64) / size)
    angle = (pos.reshape(-1, 1, 1) + c["prefix"]).double() * freq  # far positions times the fastest frequency need 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _turned(s["q"].reshape(rows, -1, size).float(), s["gains"][0], cos, sin, c["neox"])
    k = _turned(s["new_k"].reshape(rows, -1, size).float(), s["gains"][1], cos, sin, c["neox"])
    new, pos = new.reshape(-1), pos.reshape(-1)
    s["q_out"].copy_(torch.where(new[:, None], q.reshape(rows, -1).to(s["q_out"].dtype), s["q_out"]))
    table = s["table"].repeat_interleave(c["n_query"], 0)
    at = torch.gather(table, 1, (pos // page).clamp(0, table.shape[1] - 1)[:, None])[:, 0].long()
    at = torch.where(new, at, s["n_pages"])
    s["k"][at, :, pos % page] = k.to(s["k"].dtype)
    s["v"][at, :, pos % page] = s["new_v"].reshape(rows, -1, size).to(s["v"].dtype)


def _plain_attention(s):
    c = s["case"]
    B, J, H, size = c["n_seq"], c["n_query"], c["kv_heads"], c["size"]
    G = c["heads"] // H
    pos, new = _places(s)
    q = s["q"].reshape(B, J, H, G, size).float().permute(0, 2, 1, 3, 4) * size ** -0.5
    table = s["table"].clamp(min=0).long()
    k, v = (s[x][table].permute(0, 2, 1, 3, 4).reshape(B, H, -1, size).float() for x in "kv")  # [sequence, head, own position, size]
    seen = torch.arange(k.shape[2], device="cuda") <= pos[:, :, None]  # [sequence, query, own position]
    scores = torch.matmul(q.reshape(B, H, J * G, size), k.transpose(-1, -2)).reshape(B, H, J, G, -1)
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    pre = s["prefix_pages"].long()
    pk, pv = (s[x][pre].permute(1, 0, 2, 3).reshape(H, -1, size)[:, :c["prefix"]].float() for x in "kv")
    first = torch.matmul(q.permute(1, 0, 2, 3, 4).reshape(H, -1, size), pk.transpose(-1, -2)).reshape(H, B, J, G, -1).transpose(0, 1)
    top = torch.cat((scores.amax(-1, keepdim=True), first.amax(-1, keepdim=True)) if c["prefix"] else (scores.amax(-1, keepdim=True),), -1).amax(-1, keepdim=True).clamp(min=-1e30)
    scores, first = (scores - top).exp(), (first - top).exp()
    out = torch.matmul(scores.reshape(B, H, J * G, -1), v).reshape(B, H, J, G, size)
    out = out + torch.matmul(first.transpose(0, 1).reshape(H, B * J * G, -1), pv).reshape(H, B, J, G, size).transpose(0, 1)
    total = scores.sum(-1, keepdim=True) + first.sum(-1, keepdim=True)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 2, 1, 3, 4).reshape(B * J, -1)
    s["out"].copy_(torch.where(new.reshape(-1, 1), out.to(s["out"].dtype), s["out"]))


def _plain_sample(s):
    x = s["logits"].float()
    x = torch.where(x > -math.inf, x, -math.inf)  # no number: not a choice
    order = torch.sort(x, dim=1, descending=True, stable=True)
    sorted_x, top = order.values, order.values[:, :1]
    t = s["temperature"].double()[:, None]
    greedy = ~(t > 0)
    w = ((sorted_x.double() - top.double()) / torch.where(greedy, 1.0, t)).exp()
    w = torch.where(sorted_x == top, 1.0, torch.where(sorted_x > -math.inf, w, 0.0))
    rank = torch.arange(x.shape[1], device="cuda")[None]
    k, p, m = s["top_k"][:, None], s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    keep = (rank < k) | (k <= 0)
    w = torch.where(keep, w, 0.0)
    before = w.cumsum(1) - w
    keep &= ((before < p * w.sum(1, keepdim=True)) | (p >= 1)) & (w >= m)
    keep |= rank == 0
    w = torch.where(keep & ((rank == 0) | ~greedy), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order.indices, w)  # in the order of the vocabulary
    total = w.cumsum(1)
    chosen = (total > s["uniform"][:, None] * total[:, -1:]).int().argmax(1)
    s["tokens"].copy_(chosen)
    s["probs"].copy_(w.gather(1, chosen[:, None])[:, 0] / total[:, -1])


# ---- what one pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * SIZE[c["io"]] + c["rows"] * 32, "flops": 4 * n}
    past, counts = _lengths(c, 1)
    new, heads, kv, size, io, cache = int(counts.sum()), c["heads"], c["kv_heads"], c["size"], SIZE[c["io"]], SIZE[c["cache"]]
    if c["kind"] == "append":
        values = new * size
        return {"bytes": values * ((2 * heads + 2 * kv) * io + 2 * kv * cache), "flops": values * (heads + kv) * (7 if c["norm"] else 3)}
    keys = int((past + counts).sum()) + c["prefix"]
    pairs = int((counts * (past + c["prefix"]) + counts * (counts + 1) // 2).sum())
    return {"bytes": 2 * keys * kv * size * cache + 2 * new * heads * size * io, "flops": 4 * pairs * heads * size}


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] == "sample":
        tokens, probs = s["tokens"].cpu(), s["probs"].double().cpu()
        for r in range(c["rows"]):
            tokens[r], probs[r] = _exact_row(s["logits"][r].double(), s["uniform"][r].item(), *(s[n][r].item() for n in ("temperature", "top_k", "top_p", "min_p")))
        return {"tokens": tokens, "probs": probs}
    past, counts = _lengths(c, seed)
    out = {k: s[k].double() for k in ("q_out", "k", "v", "out") if k in s}
    size, page, G = c["size"], c["page"], c["heads"] // c["kv_heads"]
    table = s["table"].long()
    pre = s["prefix_pages"].long()
    flat = lambda pool, pages, n: pool[pages].double().transpose(1, 2).reshape(-1, c["kv_heads"], size)[:n]  # noqa: E731
    for i in range(c["n_seq"]):
        lo, n, m = i * c["n_query"], int(counts[i]), int(past[i])
        own_pos = torch.arange(m, m + n, device="cuda")
        q = s["q"][lo:lo + n].double().reshape(n, c["heads"], size)
        if c["kind"] == "append":
            k, v = (s[x][lo:lo + n].double().reshape(n, c["kv_heads"], size) for x in ("new_k", "new_v"))
            half = torch.arange(size // 2, device="cuda", dtype=torch.float64)
            turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), (own_pos + c["prefix"]).double()[:, None] * torch.exp(half * (-2 * math.log(10000.0) / size)))[:, None]
            for x, gain, name in ((q, s["gains"][0], "q_out"), (k, s["gains"][1], "k")):
                if gain is not None:
                    x = gain.double() * x / ((x ** 2).sum(-1, keepdim=True) / size + EPS).sqrt()
                pair = x.reshape(n, -1, 2, size // 2).transpose(2, 3) if c["neox"] else x.reshape(n, -1, size // 2, 2)
                y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
                y = (y.transpose(2, 3) if c["neox"] else y).reshape(x.shape)
                if name == "q_out":
                    out["q_out"][lo:lo + n] = y.reshape(n, -1)
                else:
                    out["k"][table[i, own_pos // page], :, own_pos % page] = y
            out["v"][table[i, own_pos // page], :, own_pos % page] = v
        else:
            used = table[i][: -(-(m + n) // page)]
            k, v = (torch.cat((flat(s[x], pre, c["prefix"]), flat(s[x], used, m + n))).repeat_interleave(G, 1) for x in "kv")
            z = torch.einsum("nhd,khd->hnk", q, k) / math.sqrt(size)
            ahead = torch.arange(k.shape[0], device="cuda")[None] > (own_pos + c["prefix"])[:, None]
            a = torch.softmax(z.masked_fill(ahead, -math.inf), -1)
            out["out"][lo:lo + n] = torch.einsum("hnk,khd->nhd", a, v).reshape(n, -1)
    if c["kind"] == "append":
        return {"q": out["q_out"], "k": out["k"][:s["n_pages"]], "v": out["v"][:s["n_pages"]]}
    return {"out": out["out"]}


def _exact_row(x, u, t, k, p, m):
    order = torch.argsort(x, descending=True, stable=True)
    if t <= 0:
        return int(order[0]), 1.0
    order = order[:k] if k > 0 else order
    share = torch.softmax(x[order] / t, 0)
    n = int(torch.searchsorted(share.cumsum(0), p * share.sum())) + 1 if p < 1 else len(order)
    order, share = order[:n], share[:n]
    order = order[share >= m * share[0]].sort().values
    share = torch.softmax(x[order] / t, 0)
    at = min(int(torch.searchsorted(share.cumsum(0), u, right=True)), len(order) - 1)
    return int(order[at]), float(share[at])
