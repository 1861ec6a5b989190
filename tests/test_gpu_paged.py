"""The paged cache's operators on device pointers (append, attention over a shared prefix and own pages) against plain forms in 64 bits.

Pool slots that no row's result may hang on hold NaN.  Half a step of a type is eps / 2 relative; u = 2^-24 is half a step of f32."""
import ctypes as C
import math

import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
GGML = {"f32": 0, "f16": 1, "bf16": 30}


@pytest.fixture(scope="module")
def L(pkg):
    from llama2_jl_b200 import _lib
    _lib.lib()
    return _lib


def dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def at(t):
    return None if t is None else t.data_ptr()


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


class Batch:
    """Pages in random order, lengths and counts as given; everything else of the pools is NaN unless `fill` puts numbers there."""

    def __init__(self, L, lengths, n_query=1, counts=None, kv=2, hs=64, page=16, prefix=0, cache="bf16", seed=0, width=None, filled=True, extra_pages=0):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.L, self.kv, self.hs, self.page, self.prefix, self.n_query, self.cache = L, kv, hs, page, prefix, n_query, cache
        self.n_seq = len(lengths)
        width = max([-(-max(n, 0) // page) for n in lengths] + [0]) if width is None else width
        pre = -(-prefix // page)
        self.n_pages = pre + self.n_seq * width + 3 + extra_pages
        order = torch.randperm(self.n_pages, generator=g, device="cuda")
        self.prefix_pages = order[:pre].to(torch.int32)
        self.table = torch.full((self.n_seq, width), -1, dtype=torch.int32, device="cuda")
        for i, n in enumerate(lengths):
            m = min(width, -(-max(n, 0) // page))
            self.table[i, :m] = order[pre + i * width:pre + i * width + m]
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
        shape = (self.n_pages, kv, page, hs)
        self.k, self.v = (torch.full(shape, float("nan"), device="cuda", dtype=dtype(cache)) for _ in "kv")
        if filled:
            for pool in (self.k, self.v):
                x = torch.randn(shape, generator=g, device="cuda").to(pool.dtype)
                for pages, n in [(self.prefix_pages, prefix)] + [(self.table[i], n) for i, n in enumerate(lengths)]:
                    for b in range(min(-(-max(n, 0) // page), len(pages))):
                        pool[pages[b], :, :min(page, n - b * page)] = x[pages[b], :, :min(page, n - b * page)]

    def structs(self):
        L = self.L
        return (L.PagedCache(dev_k=at(self.k), dev_v=at(self.v), type=GGML[self.cache], n_pages=self.n_pages, page_size=self.page, n_kv_heads=self.kv, head_size=self.hs),
                L.PagedBatch(n_seq=self.n_seq, n_query=self.n_query, dev_lengths=at(self.lengths), dev_counts=at(self.counts), dev_pages=at(self.table) or None,
                             pages_per_seq=self.table.shape[1], prefix_len=self.prefix, dev_prefix_pages=at(self.prefix_pages) if self.prefix else None))

    def new_rows(self):
        """(row, sequence, own position) of every new token."""
        out = []
        lengths = self.lengths.tolist()
        counts = [self.n_query] * self.n_seq if self.counts is None else self.counts.tolist()
        for i, (n, c) in enumerate(zip(lengths, counts)):
            c = max(0, min(c, self.n_query)) if n >= 0 else 0
            out += [(i * self.n_query + j, i, n - c + j) for j in range(c)]
        return out

    def place(self, seq, pos):
        """(page, slot) of an own position, None where it has no page."""
        if pos < 0 or pos >= self.table.shape[1] * self.page or pos >= int(self.lengths[seq]):
            return None
        page = int(self.table[seq, pos // self.page])
        return (page, pos % self.page) if 0 <= page < self.n_pages else None

    def append(self, rows):
        cache, batch = self.structs()
        self.L.check(self.L.lib().l2b_paged_append_device(C.byref(cache), C.byref(batch), C.byref(rows), stream()))

    def plan(self, q, out, heads, scale=0.0):
        import torch
        kind = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}[q.dtype]
        queries = self.L.PagedQueries(type=kind, n_heads=heads, dev_q=at(q), q_stride=q.stride(0), dev_out=at(out), out_stride=out.stride(0), scale=scale)
        cache, batch = self.structs()
        need = C.c_int64()
        self.L.check(self.L.lib().l2b_paged_attention_workspace(C.byref(cache), C.byref(batch), C.byref(queries), C.byref(need)))
        return [cache, batch, queries, torch.full((max(1, need.value // 4),), float("nan"), device="cuda")]

    def attend(self, plan):
        cache, batch, queries, w = plan
        self.L.check(self.L.lib().l2b_paged_attention_device(C.byref(cache), C.byref(batch), C.byref(queries), at(w), w.numel() * 4, stream()))


# ---- append ---------------------------------------------------------------------------------------------------------------------
def turned(x, gain, pos, base, neox, eps):
    """x [heads, hs] in f64 -> (result, |a| + |b| of each value's pair: the scale of its rounding errors)."""
    import torch
    hs = x.shape[-1]
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double()
    if base == 0:
        return x, x.abs()
    t = pos * base ** (-torch.arange(0, hs, 2, dtype=torch.float64, device=x.device) / hs)
    a, b = (x[..., :hs // 2], x[..., hs // 2:]) if neox else (x[..., 0::2], x[..., 1::2])
    y, size = (a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()), a.abs() + b.abs()
    join = (lambda p: torch.cat(p, -1)) if neox else (lambda p: torch.stack(p, -1).flatten(-2))
    return join(y), join((size, size))


@pytest.mark.parametrize("io,cache", [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f16")])
@pytest.mark.parametrize("heads,kv,hs,neox,norm,base", [(8, 2, 128, False, True, 10000.0), (3, 3, 96, True, True, 500000.0), (6, 1, 24, True, False, 10000.0), (2, 2, 8, False, True, 100.0),
                                                        (5, 5, 80, False, False, 10000.0), (4, 2, 64, True, False, 0.0), (7, 1, 40, False, True, 10000.0)])
def test_append(L, io, cache, heads, kv, hs, neox, norm, base):
    import torch
    lengths, counts = [37, -1, 3, 0, 16, 5, 70], [3, 3, 5, 0, 1, 2, 4]  # (a sequence that sits out, more rows than positions, none, one)
    b = Batch(L, lengths, n_query=4, counts=counts, kv=kv, hs=hs, page=8, prefix=100003, cache=cache, seed=hs, filled=False, width=8)  # (70: beyond the table)
    b.table[0, 2] = -1  # a page that is none, and one that does not exist
    b.table[5, 0] = b.n_pages
    g, t = torch.Generator(device="cuda").manual_seed(1), dtype(io)
    width, rows = (heads + 2 * kv) * hs + 8, b.n_seq * 4  # (rows further apart than they are long)
    qkv = (torch.randn((rows, width), generator=g, device="cuda") * 2).to(t)
    q, k, v = qkv[:, :heads * hs], qkv[:, heads * hs:(heads + kv) * hs], qkv[:, (heads + kv) * hs:(heads + 2 * kv) * hs]
    q_out = torch.full((rows, heads * hs + 16), 7.0, device="cuda", dtype=t)
    gains = [(1 + 0.2 * torch.randn(hs, generator=g, device="cuda")) if norm else None for _ in range(2)]
    eps = 1e-5
    b.append(L.PagedRows(type=GGML[io], n_heads=heads, dev_q=at(q), dev_k=at(k), dev_v=at(v), q_stride=width, k_stride=width, v_stride=width, dev_q_out=at(q_out), q_out_stride=heads * hs + 16,
                         dev_q_gain=at(gains[0]), dev_k_gain=at(gains[1]), eps=eps, rope_freq_base=base, rope_is_neox=int(neox)))
    want_k, want_v, untouched = torch.full_like(b.k, float("nan")), torch.full_like(b.v, float("nan")), torch.ones(rows, dtype=torch.bool)
    # u per value: the norm's sum (at most 24 additions, half of it after the root), root, division and two products 18; the angle and its sine
    # and cosine 6, the rotation's products and sum 3: less than 32
    for row, seq, pos in b.new_rows():
        untouched[row] = False
        want, size = turned(q[row].double().view(heads, hs), gains[0], 100003 + pos, base, neox, eps)
        err = (q_out[row, :heads * hs].double().view(heads, hs) - want).abs()
        assert (err <= torch.finfo(t).eps / 2 * (want.abs() + 32 * U * size) + 32 * U * size + 1e-30).all(), (row, err.max())
        place = b.place(seq, pos)
        if place:
            want, size = turned(k[row].double().view(kv, hs), gains[1], 100003 + pos, base, neox, eps)
            got = b.k[place[0], :, place[1]]
            tiny = 2.0 ** -25 if cache == "f16" else 0.0  # half a step of f16 numbers below 2^-14
            assert ((got.double() - want).abs() <= torch.finfo(got.dtype).eps / 2 * (want.abs() + 32 * U * size) + 32 * U * size + tiny).all()
            want_k[place[0], :, place[1]] = got
            want_v[place[0], :, place[1]] = v[row].view(kv, hs).to(want_v.dtype)
    assert torch.equal(b.k.isnan(), want_k.isnan()) and torch.equal(b.v.nan_to_num(9), want_v.nan_to_num(9))  # nothing else is written
    assert (q_out[:, heads * hs:] == 7).all() and (q_out[untouched.cuda()] == 7).all()


def test_append_in_place_without_queries_and_far_positions(L):
    import torch
    b = Batch(L, [3], n_query=3, kv=2, hs=64, page=16, prefix=1, cache="bf16", filled=False)
    b.prefix = 0x7fffffff - 16  # (its pages are not read here)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn((3, 4 * 64), generator=g, device="cuda")
    kv = torch.randn((3, 2 * 64), generator=g, device="cuda")
    before = q.clone()
    b.append(L.PagedRows(type=0, n_heads=4, dev_q=at(q), dev_k=at(kv), dev_v=at(kv), q_stride=256, k_stride=128, v_stride=128, dev_q_out=at(q), q_out_stride=256, rope_freq_base=10000.0))
    for r in range(3):
        want, size = turned(before[r].double().view(4, 64), None, 0x7fffffff - 16 + r, 10000.0, False, 0)
        # the position times the frequency is off by half a step of 64 bits: up to 2^31 / 2 pi turns * 2^-53, in radians 2^31 * 2^-53 = 4 u, and the frequency by as much,
        # here and in the reference
        assert ((q[r].double().view(4, 64) - want).abs() <= 48 * U * size).all()
    was = b.k.clone()
    b.append(L.PagedRows(type=0, n_heads=0, dev_q=None, dev_k=at(kv), dev_v=at(kv), k_stride=128, v_stride=128, rope_freq_base=10000.0))
    assert torch.equal(was.nan_to_num(9), b.k.nan_to_num(9))


@pytest.mark.parametrize("n_seq,n_query", [(1, 1), (3, 500), (300, 1), (1, 3001), (2500, 1)])
def test_append_of_few_and_many_rows(L, n_seq, n_query):
    """Every grid shape: all rows land, once, whatever the tokens of a block."""
    import torch
    kv, hs, heads = 2, 64, 6
    b = Batch(L, [n_query + i % 5 for i in range(n_seq)], n_query=n_query, kv=kv, hs=hs, page=64, cache="f16", filled=False)
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = n_seq * n_query
    q, k, v = (torch.randn((rows, h * hs), generator=g, device="cuda").half() for h in (heads, kv, kv))
    q_out = torch.zeros_like(q)
    b.append(L.PagedRows(type=1, n_heads=heads, dev_q=at(q), dev_k=at(k), dev_v=at(v), q_stride=heads * hs, k_stride=kv * hs, v_stride=kv * hs, dev_q_out=at(q_out), q_out_stride=heads * hs))
    assert torch.equal(q, q_out)  # (no norm, no rotation)
    seq = torch.arange(rows, device="cuda") // n_query
    pos = b.lengths.long()[seq] - n_query + torch.arange(rows, device="cuda") % n_query
    page = b.table.long()[seq, pos // 64]
    assert torch.equal(b.k[page, :, pos % 64].reshape(rows, -1), k) and torch.equal(b.v[page, :, pos % 64].reshape(rows, -1), v)
    assert int((~b.k.isnan()).sum()) == rows * kv * hs


# ---- attention ------------------------------------------------------------------------------------------------------------------
def attention_reference(b, q, heads, scale=0.0):
    """{row: (result [heads, hs], tolerance [heads, hs])} in f64."""
    import torch
    scale = scale or b.hs ** -0.5
    G, out = heads // b.kv, {}
    half = torch.finfo(q.dtype).eps / 2
    for row, seq, pos in b.new_rows():
        places = []
        for pages, n in ((b.prefix_pages, b.prefix), (b.table[seq], min(pos + 1, b.table.shape[1] * b.page, int(b.lengths[seq])))):
            n = max(n, 0)
            i = torch.arange(n, device="cuda")
            page = pages.long()[i // b.page] if n else i
            fine = (page >= 0) & (page < b.n_pages)
            places.append((page[fine], i[fine] % b.page))
        page, slot = (torch.cat(x) for x in zip(*places))
        k, v = (pool[page, :, slot].double().repeat_interleave(G, 1) for pool in (b.k, b.v))  # [n, heads, hs]
        x = q[row, :heads * b.hs].double().view(heads, b.hs)
        if not len(page):
            out[row] = (torch.zeros_like(x), torch.zeros_like(x))
            continue
        z = torch.einsum("hd,nhd->hn", x, k) * scale
        w = torch.softmax(z, -1)
        o, size = torch.einsum("hn,nhd->hd", w, v), torch.einsum("hn,nhd->hd", w, v.abs())
        # Scores: at most 24 products of 16 are added up (three terms of 8), each sum off by a step of f32 at most, 24 * 2^-23 < 2^-18 of their absolute size.
        ds = 2.0 ** -18 * (torch.einsum("hd,nhd->hn", x.abs(), k.abs()) * abs(scale)).amax(-1)
        # Weights: rounded to the cache's type once for rows of that type; for f32 rows three terms of bf16 or two of f16, half a step to that power (f16: or
        # 2^-25 of the largest weight, a number below 2^-14); sums: a step of f32 per 16 keys.
        weights = half if q.dtype != torch.float32 else (torch.finfo(b.k.dtype).eps / 2) ** (3 if b.cache == "bf16" else 2)
        tiny = (2.0 ** -25 * v.abs().sum(0)) if b.cache == "f16" else 0.0
        steps = (len(page) / 16 + 16) * 2.0 ** -23
        tol = (weights + ds[:, None] + steps) * size + tiny
        out[row] = (o, tol + half * (o.abs() + tol) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0))
    return out


def check_attention(b, q, heads, scale=0.0, pad=0):
    import torch
    out = torch.full((q.shape[0], heads * b.hs + pad), 7.0, device="cuda", dtype=q.dtype)
    b.attend(b.plan(q, out, heads, scale))
    want = attention_reference(b, q, heads, scale)
    for row in range(q.shape[0]):
        if row not in want:
            assert (out[row] == 7).all(), row  # padding and sequences that sit out
        else:
            o, tol = want[row]
            err = (out[row, :heads * b.hs].double().view(heads, b.hs) - o).abs()
            assert (err <= tol).all(), (row, float((err - tol).max()), float(err.max()))
    assert (out[:, heads * b.hs:] == 7).all()
    return out


def queries(b, heads, io, seed=5, scale=2.0, pad=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((b.n_seq * b.n_query, heads * b.hs + pad), generator=g, device="cuda") * scale).to(dtype(io))


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")]


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("heads,kv,hs,page", [(8, 2, 128, 16), (4, 4, 64, 8), (6, 2, 96, 64), (7, 1, 80, 32), (2, 2, 8, 128), (16, 1, 24, 8), (20, 1, 48, 256), (3, 3, 40, 1024)])
@pytest.mark.parametrize("prefix", [0, 1, 70, 300])
def test_attention(L, io, cache, heads, kv, hs, page, prefix):
    """Single tokens: lengths around the tiles' ends, none, sitting out; rows of q and out further apart than they are long."""
    b = Batch(L, [1, 0, 63, 64, 65, -1, 200, 17, 129], kv=kv, hs=hs, page=page, prefix=prefix, cache=cache, seed=hs + prefix)
    check_attention(b, queries(b, heads, io, pad=8), heads, pad=16)


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("n_query,heads,kv,hs", [(2, 8, 2, 128), (5, 6, 2, 64), (9, 4, 1, 96), (70, 3, 3, 64)])
@pytest.mark.parametrize("prefix", [0, 130])
def test_attention_of_several_new_tokens(L, io, cache, n_query, heads, kv, hs, prefix):
    """Causal among the new tokens; padded rows; fewer positions than new tokens (the first ones see the prefix alone, or nothing)."""
    lengths = [n_query, 100, n_query + 61, 3, 150, -5, 0]
    counts = [n_query, 1, n_query - 1, n_query, 0, 2, 1]
    b = Batch(L, lengths, n_query=n_query, counts=counts, kv=kv, hs=hs, page=16, prefix=prefix, cache=cache, seed=n_query)
    check_attention(b, queries(b, heads, io), heads)


@pytest.mark.parametrize("prefix", [0, 40])
def test_pages_that_are_none(L, prefix):
    """Entries outside the pool anywhere in the tables: their positions do not count."""
    b = Batch(L, [100, 64, 9], kv=2, hs=64, page=8, prefix=prefix, cache="bf16")
    b.table[0, 0], b.table[0, 5], b.table[0, 12] = -1, b.n_pages, -(2 ** 31)
    b.table[1, 3], b.table[2, :] = 2 ** 31 - 1, -1
    if prefix:
        b.prefix_pages[2] = -7
    check_attention(b, queries(b, 4, "bf16"), 4)


def test_lengths_beyond_the_table(L):
    b = Batch(L, [5000, 32, 33], kv=1, hs=64, page=16, width=2, cache="f16")
    check_attention(b, queries(b, 2, "f16"), 2)
    b = Batch(L, [5, 1], kv=1, hs=64, page=16, width=0, prefix=20, cache="f16")  # no own pages at all
    check_attention(b, queries(b, 2, "f16"), 2)


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_a_later_token_does_not_reach_an_earlier_one(L, io):
    """Keys and values that are no numbers at the last new token's position: only its own result is lost."""
    import torch
    for bad in (float("nan"), float("inf")):
        b = Batch(L, [37], n_query=3, kv=1, hs=64, page=16, prefix=10)
        q = queries(b, 4, io)
        clean = check_attention(b, q, 4)
        page, slot = b.place(0, 36)
        b.k[page, :, slot] = bad
        b.v[page, :, slot] = bad
        out = torch.zeros_like(clean)
        b.attend(b.plan(q, out, 4))
        want = attention_reference(b, q, 4)
        for row in (0, 1):
            assert ((out[row].double().view(4, 64) - want[row][0]).abs() <= want[row][1]).all()
        assert not torch.isfinite(out[2]).any()


def test_scores_that_are_no_numbers_show(L):
    """A query of NaN gives NaN, not zeros, and leaves the other rows alone; large scores saturate without overflow."""
    import torch
    b = Batch(L, [50, 200], kv=1, hs=64, page=16)
    q = queries(b, 2, "bf16")
    q[0, :64] = float("nan")
    out = torch.zeros_like(q)
    b.attend(b.plan(q, out, 2))
    assert out[0, :64].isnan().all() and torch.isfinite(out[0, 64:]).all() and torch.isfinite(out[1]).all()
    check_attention(b, queries(b, 2, "bf16", scale=300.0), 2)
    check_attention(b, queries(b, 2, "f32", scale=300.0), 2)


@pytest.mark.parametrize("scale", [1e-20, 1e30])
def test_f32_queries_over_f16_keys_of_any_size(L, scale):
    """f32 rows may lie outside f16's range: their terms are taken behind a power of two."""
    b = Batch(L, [70, 3], kv=1, hs=64, page=16, cache="f16")
    check_attention(b, queries(b, 2, "f32", scale=scale), 2, scale=0.3 / scale)


@pytest.mark.parametrize("heads", [2, 40, 300])
@pytest.mark.parametrize("scale", [0.05, -0.2])
def test_scales(L, scale, heads):
    b = Batch(L, [70, 3], kv=1, hs=64, page=16, prefix=209)
    check_attention(b, queries(b, heads, "bf16"), heads, scale=scale)


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 512, 1024])
def test_prefixes_in_pages_of_every_size(L, page, io, cache):
    """Many rows on one prefix: pages smaller and larger than a tile of keys, the prefix's end anywhere in the last one, a hole in the middle."""
    for prefix, heads in ((page, 20), (2 * page + 1, 130), (3 * page - 1, 300), (1500, 64)):
        b = Batch(L, [5, 0], kv=2, hs=72, page=page, prefix=prefix, cache=cache, seed=prefix)
        if prefix == 3 * page - 1:
            b.prefix_pages[1] = -1
        check_attention(b, queries(b, heads, io), heads)


def test_sequences_that_share_pages_of_their_own(L):
    """The same pages in several rows of the table."""
    b = Batch(L, [40, 40, 33], kv=2, hs=64, page=16, prefix=20)
    b.table[1:] = b.table[0]
    check_attention(b, queries(b, 4, "bf16"), 4)


def test_first_calls_in_a_capture(pkg):
    """A process whose first calls are captured ones."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = """
import sys
sys.path[:0] = [%r, %r]
import __graft_entry__ as g
g.load_package()
from llama2_jl_b200 import _lib as L
import ctypes as C, torch, test_gpu_paged as T
b = T.Batch(L, [60, 200, 1, 90], kv=2, hs=128, page=16, prefix=200)
q = T.queries(b, 32, "bf16")
out, plan = torch.zeros_like(q), None
plan = b.plan(q, out, 32)
x, u, tokens = torch.zeros((3, 5000), device="cuda"), torch.full((3,), 0.5, dtype=torch.float64, device="cuda"), torch.full((3,), -7, dtype=torch.int32, device="cuda")
a = L.Sampling(type=0, n_rows=3, vocab=5000, dev_logits=T.at(x), stride=5000, dev_uniform=T.at(u), dev_tokens=T.at(tokens))
rows = torch.ones((4, 256), device="cuda").bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    b.append(L.PagedRows(type=30, dev_k=T.at(rows), dev_v=T.at(rows), k_stride=256, v_stride=256, rope_freq_base=1e4))
    b.attend(plan)
    L.check(L.lib().l2b_sample_device(C.byref(a), T.stream()))
graph.replay()
torch.cuda.synchronize()
for r, (o, tol) in T.attention_reference(b, q, 32).items():
    assert ((out[r].double().view(32, 128) - o).abs() <= tol).all()
assert tokens.tolist() == [2500] * 3
print("done")
""" % (here, os.path.dirname(here))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("n_seq,prefix,most,heads,kv,hs", [(1, 0, 5000, 8, 2, 128), (1, 3000, 1, 8, 2, 128), (70, 900, 90, 8, 2, 64), (40, 0, 2000, 4, 4, 96), (3, 2500, 1500, 32, 1, 64)])
@pytest.mark.parametrize("io,cache", [("bf16", "bf16"), ("f32", "f16")])
def test_long_and_many(L, n_seq, prefix, most, heads, kv, hs, io, cache):
    """Items that many blocks share, blocks that share many items."""
    import numpy as np
    lengths = np.random.default_rng(n_seq).integers(1, most + 1, n_seq).tolist()
    b = Batch(L, lengths, kv=kv, hs=hs, page=64, prefix=prefix, cache=cache, seed=9)
    check_attention(b, queries(b, heads, io), heads)


@pytest.mark.parametrize("prefix", [0, 500])
def test_offsets_beyond_32_bits(L, prefix):
    """A pool of more than 2^32 values; the pages in use lie at its end."""
    import torch
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    b = Batch(L, [100, 33], kv=8, hs=128, page=64, prefix=prefix)
    small_k, small_v, n = b.k, b.v, b.n_pages
    b.n_pages = 66000 + n
    assert b.n_pages * 8 * 64 * 128 > 1 << 32
    b.k, b.v = (torch.empty((b.n_pages, 8, 64, 128), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    b.k[66000:], b.v[66000:] = small_k, small_v
    b.table = torch.where(b.table >= 0, b.table + 66000, -1)
    b.prefix_pages = b.prefix_pages + 66000
    check_attention(b, queries(b, 8, "bf16"), 8)
    rows = torch.randn((2, 8 * 128), device="cuda").bfloat16()
    b.append(L.PagedRows(type=30, dev_k=at(rows), dev_v=at(rows), k_stride=1024, v_stride=1024))
    for i, n in enumerate([100, 33]):
        page, slot = b.place(i, n - 1)
        assert torch.equal(b.v[page, :, slot].reshape(-1), rows[i])


@pytest.mark.parametrize("io,prefix", [("bf16", 0), ("bf16", 200), ("f32", 200)])
def test_same_bits_twice_and_in_graphs(L, io, prefix):
    """A captured call reads lengths, pages and queries when it runs; two graphs with workspaces of their own may run side by side."""
    import torch
    b = Batch(L, [60, 200, 1, 90], kv=2, hs=128, page=16, prefix=prefix, width=20)
    q = queries(b, 8, io)
    eager = check_attention(b, q, 8)
    assert torch.equal(eager, check_attention(b, q, 8))
    outs, graphs, plans = [torch.zeros_like(eager) for _ in range(2)], [], []
    side = [torch.cuda.Stream() for _ in range(2)]
    for o, s in zip(outs, side):
        plan = b.plan(q, o, 8)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            b.attend(plan)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                b.attend(plan)
        graphs.append(g)
        plans.append(plan)
    torch.cuda.synchronize()
    for trial in range(3):
        for o in outs:
            o.fill_(7)
        b.lengths.copy_(torch.tensor([[60, 200, 1, 90], [17, 100, -1, 64], [1, 0, 1, 33]][trial], device="cuda", dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, side):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        want = torch.full_like(eager, 7)
        b.attend(b.plan(q, want, 8))
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_nothing_to_do(L):
    import torch
    b = Batch(L, [5, 6], kv=1, hs=64, page=16)
    q = queries(b, 2, "bf16")
    out = torch.full_like(q, 7)
    plan = b.plan(q, out, 2)
    plan[1].n_seq = 0
    b.attend(plan)
    cache, batch = b.structs()
    batch.n_seq = 0
    L.check(L.lib().l2b_paged_append_device(C.byref(cache), C.byref(batch), C.byref(L.PagedRows(type=30, dev_k=at(q), dev_v=at(q), k_stride=128, v_stride=128)), stream()))
    torch.cuda.synchronize()
    assert (out == 7).all()


def test_a_workspace_that_is_too_small_is_refused(L):
    import torch
    b = Batch(L, [5, 6], kv=1, hs=64, page=16, prefix=20)
    q = queries(b, 2, "bf16")
    plan = b.plan(q, torch.zeros_like(q), 2)
    lib, (cache, batch, qs, w) = L.lib(), plan
    assert lib.l2b_paged_attention_device(C.byref(cache), C.byref(batch), C.byref(qs), at(w), w.numel() * 4 - 4, None) == 1
    assert lib.l2b_paged_attention_device(C.byref(cache), C.byref(batch), C.byref(qs), None, w.numel() * 4, None) == 1
    assert lib.l2b_paged_attention_device(C.byref(cache), C.byref(batch), C.byref(qs), at(w) + 8, w.numel() * 4, None) == 1
    assert "workspace" in lib.l2b_last_error_string().decode()


def test_decode_steps_with_append_attention_and_sampling(L):
    """Four steps of a small batch as a server runs them: rows into the pages, attention, a product with the vocabulary's rows, the next tokens; against
    the same steps in 64 bits over what the cache then holds."""
    import torch
    heads, kv, hs, vocab, n_seq, prefix, steps = 8, 2, 64, 1000, 5, 37, 4
    start = [0, 3, 15, 16, 40]
    g = torch.Generator(device="cuda").manual_seed(11)
    b = Batch(L, start, kv=kv, hs=hs, page=16, prefix=prefix, width=4)
    for i, n in enumerate(start):  # a page for what is to come
        for j in range(4):
            if int(b.table[i, j]) < 0:
                used = set(b.table.flatten().tolist()) | set(b.prefix_pages.tolist())
                b.table[i, j] = next((p for p in range(b.n_pages) if p not in used), -1)
    words = torch.randn((vocab, heads * hs), generator=g, device="cuda")
    gain = 1 + 0.1 * torch.randn(hs, generator=g, device="cuda")
    out, tokens, probs = torch.zeros((n_seq, heads * hs), device="cuda"), torch.zeros(n_seq, dtype=torch.int32, device="cuda"), torch.zeros(n_seq, device="cuda")
    logits = torch.zeros((n_seq, vocab), device="cuda")
    uniform = torch.rand(n_seq, generator=g, device="cuda", dtype=torch.float64)
    top_k = torch.full((n_seq,), 20, dtype=torch.int32, device="cuda")
    for step in range(steps):
        b.lengths += 1
        qkv = torch.randn((n_seq, (heads + 2 * kv) * hs), generator=g, device="cuda")
        q, k, v = qkv[:, :heads * hs], qkv[:, heads * hs:(heads + kv) * hs], qkv[:, (heads + kv) * hs:]
        before, w = q.clone(), qkv.stride(0)
        b.append(L.PagedRows(type=0, n_heads=heads, dev_q=at(q), dev_k=at(k), dev_v=at(v), q_stride=w, k_stride=w, v_stride=w, dev_q_out=at(q), q_out_stride=w, dev_q_gain=at(gain), dev_k_gain=at(gain),
                             eps=1e-6, rope_freq_base=10000.0))
        b.attend(b.plan(q, out, heads))
        torch.matmul(out, words.T, out=logits)
        L.check(L.lib().l2b_sample_device(C.byref(L.Sampling(type=0, n_rows=n_seq, vocab=vocab, dev_logits=at(logits), stride=vocab, dev_top_k=at(top_k), dev_uniform=at(uniform), dev_tokens=at(tokens),
                                                            dev_probs=at(probs))), stream()))
        turned_q = torch.zeros((n_seq, heads * hs), dtype=torch.float64, device="cuda")
        for row, seq, pos in b.new_rows():
            want, size = turned(before[row].double().view(heads, hs), gain, prefix + pos, 10000.0, False, 1e-6)
            assert ((q[row].double().view(heads, hs) - want).abs() <= 33 * U * size).all()
            turned_q[row] = want.flatten()
            page, slot = b.place(seq, pos)
            want, size = turned(k[row].double().view(kv, hs), gain, prefix + pos, 10000.0, False, 1e-6)
            assert ((b.k[page, :, slot].double() - want).abs() <= 2.0 ** -8 * (want.abs() + 32 * U * size) + 32 * U * size).all()
        for row, (o, tol) in attention_reference(b, q, heads).items():
            assert ((out[row].double().view(heads, hs) - o).abs() <= tol).all()
        for row in range(n_seq):
            x = logits[row].double()
            order = torch.argsort(x, descending=True, stable=True)[:20].sort().values
            share = torch.softmax(x[order], 0)
            i = int((share.cumsum(0) > float(uniform[row])).int().argmax())
            assert int(tokens[row]) == int(order[i]) and math.isclose(float(probs[row]), float(share[i]), rel_tol=1e-6)
