"""The paged operators where rounding, range and size can spoil a result without showing in random data: against definitions in 64 bits, with bounds that a lost
term, a lost bit or a wrapped place would break.  U, eps and the tolerances' names as in test_gpu_paged.py."""
import ctypes as C

import pytest

from test_gpu_paged import GGML, TYPES, Batch, at, dtype, queries, stream  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(pkg):
    from llama2_jl_b200 import _lib
    _lib.lib()
    return _lib


def half(t):
    import torch
    return torch.finfo(t).eps / 2


def keys_of(b, seq, pos):
    """Keys and values [n, kv, hs] in f64 that the token at own position `pos` sees."""
    import torch
    places = []
    for pages, n in ((b.prefix_pages, b.prefix), (b.table[seq], pos + 1)):
        i = torch.arange(n, device="cuda")
        places.append((pages.long()[i // b.page] if n else i, i % b.page))
    page, slot = (torch.cat(x) for x in zip(*places))
    return b.k[page, :, slot].double(), b.v[page, :, slot].double()


def attended(b, q, heads, scale=0.0):
    import torch
    out = torch.full_like(q, 7.0)
    b.attend(b.plan(q, out, heads, scale))
    return out


@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("lengths,prefix,heads,kv,hs", [([301, 64, 17], 0, 4, 2, 64), ([300, 5], 0, 16, 1, 128), ([9, 1], 500, 8, 2, 96), ([9, 1], 500, 64, 2, 96), ([40] * 9, 700, 40, 1, 128)])
def test_rows_of_16_bits_are_rounded_once(L, io, lengths, prefix, heads, kv, hs):
    """What leaves is the 64-bit result rounded once, but for errors of 32-bit size: softmax weights are not cut to 8 or 11 bits on the way.

    Scores: 8 products of 16, the sums off by a step of f32 each, 8 * 2^-23 = 2^-20 of their absolute size.  Weights: two terms; bf16's first is cut to 8 bits (2^-7 is
    left at most) and the second half a step of that, 2^-15; f16's are half a step squared, 2^-22, or 2^-25 of the largest weight.  Sums: two steps per 16 keys."""
    import torch
    b = Batch(L, lengths, kv=kv, hs=hs, page=16, prefix=prefix, cache=io, seed=hs + heads)
    q = queries(b, heads, io)
    out = attended(b, q, heads)
    t = dtype(io)
    for row, seq, pos in b.new_rows():
        k, v = (x.repeat_interleave(heads // kv, 1) for x in keys_of(b, seq, pos))
        x = q[row].double().view(heads, hs)
        w = torch.softmax(torch.einsum("hd,nhd->hn", x, k) * hs ** -0.5, -1)
        ds = 2.0 ** -20 * (torch.einsum("hd,nhd->hn", x.abs(), k.abs()) * hs ** -0.5).amax(-1)[:, None]
        want, size = torch.einsum("hn,nhd->hd", w, v), torch.einsum("hn,nhd->hd", w, v.abs())
        tol = ((2.0 ** -15 if io == "bf16" else 2.0 ** -22) + ds + (len(k) / 8 + 16) * 2.0 ** -23) * size + (2.0 ** -25 * v.abs().sum(0) if io == "f16" else 0.0)
        err = (out[row].double().view(heads, hs) - want).abs()
        least = 2.0 ** -25 if io == "f16" else 0.0
        assert (err <= tol + half(t) * (want.abs() + tol) + least).all(), (row, float((err / (half(t) * want.abs() + tol)).max()))


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("own,prefix,heads", [(8001, 0, 4), (1, 8000, 4), (1, 8000, 48)])
@pytest.mark.parametrize("log2_rest", [-7, -10, -12])
def test_one_key_has_nearly_all_of_the_mass(L, io, own, prefix, heads, log2_rest):
    """A key that every query asks for, whose value is zero, in front of 8 000 others that share 2^log2_rest of its mass: the result is what those others say,
    and weights of 2^-20 to 2^-25 of the largest must keep their bits.

    Weights in two f16 terms: off by 2^-22 relative, or by half a step of 2^-24 where the largest is 2^15 (own positions), 2^14 (a prefix, f32 rows) or 2^9 at least
    (a prefix, f16 rows): 2^-40, 2^-39 or 2^-34 of it.  Such errors of 8 000 keys are independent and evenly spread: the deviation of their sum is that / sqrt(3) *
    sqrt(sum v^2), and six of those are allowed."""
    import torch
    hs, n = 64, own + prefix
    b = Batch(L, [own], kv=1, hs=hs, page=64, prefix=prefix, cache="f16", seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    flat = (lambda pages, pool, count: [(int(pages[i // 64]), i % 64) for i in range(count)])
    places = flat(b.prefix_pages, b.k, prefix) + flat(b.table[0], b.k, own)
    page, slot = (torch.tensor(x, device="cuda") for x in zip(*places))
    # scores: q = (1, 0, ..), so a key's first value is its score at scale 1
    k = torch.randn((n, hs), generator=g, device="cuda").half()
    k[:, 0] = (torch.rand(n, generator=g, device="cuda") * 0.5).half()
    k[0, 0] = 0.0
    v = (1 + torch.rand((n, hs), generator=g, device="cuda")).half()
    v[0] = 0
    k[0, 0] = float(torch.logsumexp(k[1:, 0].double(), 0)) - log2_rest * 0.6931471805599453
    b.k[page, 0, slot], b.v[page, 0, slot] = k, v
    q = torch.zeros((1, heads * hs), device="cuda", dtype=dtype(io))
    q[0, ::hs] = 1
    out = attended(b, q, heads, 1.0)
    z = k[:, 0].double()
    w = torch.softmax(z, 0)
    want = w @ v.double()
    # scores are exact; the exponent's argument (up to 31 in base 2) is off by half a step of 2^-19, the exponential by 2^-22; sums: a step per 16 keys
    tol = want * (2.0 ** -20 + 2.0 ** -22 + 2.0 ** -22 + (n / 16 + 16) * 2.0 ** -23)
    tol = tol + (2.0 ** -40 if not prefix else 2.0 ** -39 if io == "f32" else 2.0 ** -34) * 6 / 3 ** 0.5 * (v.double() ** 2).sum(0).sqrt()
    tol = tol + half(q.dtype) * want + (2.0 ** -25 if io == "f16" else 0.0)
    err = (out.double().view(heads, hs) - want).abs()
    assert (err <= tol).all(), float((err / want).max())


@pytest.mark.parametrize("heads,own,prefix", [(4, 90, 0), (48, 1, 90)])
def test_f32_queries_of_many_sizes_over_f16_keys(L, heads, own, prefix):
    """One value of the query 2^17 times as large as the others, where the keys are zero: the others' bits count.

    A query's value in two f16 terms is off by 2^-22 relative, or by 2^-39 of the row's largest."""
    import torch
    hs = 64
    b = Batch(L, [own], kv=1, hs=hs, page=16, prefix=prefix, cache="f16", seed=5)
    b.k *= 30
    b.k[..., 0] = 0
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn((1, heads, hs), generator=g, device="cuda") * 0.05
    q[..., 0] = 8000.0
    q = q.view(1, -1)
    out = attended(b, q, heads)
    k, v = (x[:, 0] for x in keys_of(b, 0, own - 1))
    x = q.double().view(heads, hs)
    w = torch.softmax(x @ k.T * hs ** -0.5, -1)
    want, size = w @ v, w @ v.abs()
    ds = ((x.abs() * 2.0 ** -18 + 2.0 ** -39 * 8000) @ k.abs().T * hs ** -0.5).amax(-1)[:, None]  # (2^-18: terms and sums, as for every score)
    tol = (ds + 2.0 ** -22 + (len(k) / 16 + 16) * 2.0 ** -23) * size + 2.0 ** -24 * want.abs()
    err = (out.double().view(heads, hs) - want).abs()
    assert (err <= tol).all(), float((err - tol).max())


def terms(x, t, n):
    """x in f64 as the sum of n terms of the type t."""
    import torch
    left, total = x.clone(), torch.zeros_like(x)
    for _ in range(n):
        y = left.to(t).double()
        total, left = total + y, left - y
    return total


@pytest.mark.parametrize("cache", ["bf16", "f16"])
@pytest.mark.parametrize("own,prefix,heads", [(2, 0, 8), (2, 0, 64), (1, 1, 64), (0, 2, 64)])
def test_every_term_of_f32_rows_counts(L, cache, own, prefix, heads):
    """Two keys, a power of two and zero, queries with one value: the score q * 2^j is exact, the result is w / (1 + w) times a value of one, w = exp(-score).

    Score about 8: the result hangs on the query's last bits.  Score about 1: on the weight's."""
    import torch
    hs, t = 64, dtype(cache)
    full = 3 if cache == "bf16" else 2
    for j, bound_of_terms in ((3, "query"), (0, "weight")):
        b = Batch(L, [own], kv=1, hs=hs, page=8, prefix=prefix, cache=cache, width=1)
        for pool in (b.k, b.v):
            pool.zero_()
        where = [(b.prefix_pages, i) for i in range(prefix)] + [(b.table[0], i) for i in range(own)]
        (p0, s0), (p1, s1) = [(int(pages[0]), i) for pages, i in where]
        b.k[p0, 0, s0, 5] = 2.0 ** j  # the dominant key, with a value of zero
        b.v[p1, 0, s1] = 1
        g = torch.Generator(device="cuda").manual_seed(7)
        q = torch.zeros((1, heads, hs), device="cuda")
        q[0, :, 5] = 1 + torch.rand(heads, generator=g, device="cuda")
        out = attended(b, q.view(1, -1), heads, 1.0).double().view(heads, hs)
        score = q[0, :, 5].double() * 2.0 ** j
        w = torch.exp(-score)
        want = (w / (1 + w))[:, None]
        # relative: the score off by a step of f32 for its scale and one for each of its sums (4), the exponent's argument (below 32, 4 in base 2) by half a step,
        # the exponential by 2^-22, three terms by 2^-24 (two of f16: 2^-22, or half a step of 2^-24 where the largest weight is 2^14 at least), sum, quotient and their
        # rounding by 2^-22
        tol = score * 5 * 2.0 ** -23 + (2.0 ** -20 if j else 2.0 ** -23) + 3 * 2.0 ** -22 + (2.0 ** -39 / w if cache == "f16" else 0.0)
        assert ((out - want).abs() <= tol[:, None] * want).all(), (bound_of_terms, float(((out - want).abs() / want).max()))
        # a term fewer would not pass
        if bound_of_terms == "query":
            lost = torch.exp(-terms(q[0, :, 5].double(), t, full - 1) * 2.0 ** j)
            lost = lost / (1 + lost)
        else:
            lost = terms(w, t, full - 1) / (1 + w)
        assert ((lost - want[:, 0]).abs() > 1.5 * tol * want[:, 0]).any()


@pytest.mark.parametrize("heads,kv,hs,neox", [(4, 2, 64, False), (4, 2, 64, True), (3, 1, 40, False), (3, 1, 40, True)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_without_rotation_leaves_neighbours_alone(L, heads, kv, hs, neox, norm):
    """rope_freq_base 0: every value comes from its own place; infinities and values that are no numbers reach no pair's other half."""
    import torch
    b = Batch(L, [3, 20], kv=kv, hs=hs, page=8, cache="bf16", filled=False)
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k = (torch.randn((2, n, hs), generator=g, device="cuda") for n in (heads, kv))
    v = torch.randn((2, kv * hs), generator=g, device="cuda")
    for x in (q, k):
        x[0, 0, 6], x[1, 0, 7] = float("inf"), -float("inf")
        if not norm:
            x[0, 0, hs // 2 + 3] = float("nan")
    q_out = torch.zeros_like(q)
    gain = (1 + 0.2 * torch.randn(hs, generator=g, device="cuda")) if norm else None
    b.append(L.PagedRows(type=0, n_heads=heads, dev_q=at(q), dev_k=at(k), dev_v=at(v), q_stride=heads * hs, k_stride=kv * hs, v_stride=kv * hs, dev_q_out=at(q_out), q_out_stride=heads * hs,
                         dev_q_gain=at(gain), dev_k_gain=at(gain), eps=1e-6, rope_is_neox=int(neox)))
    for i, n in enumerate((3, 20)):
        page, slot = b.place(i, n - 1)
        for x, got, bits in ((q, q_out[i], 0), (k, b.k[page, :, slot], 2.0 ** -8)):
            want = x[i].double()
            if norm:
                want = want / torch.sqrt((want * want).mean(-1, keepdim=True) + 1e-6) * gain.double()
            got = got.double()
            fine = want.isfinite()
            assert torch.equal(got[~fine].isnan(), want[~fine].isnan()) and torch.equal(got[~fine].nan_to_num(9), want[~fine].nan_to_num(9))
            assert ((got[fine] - want[fine]).abs() <= (bits + 32 * 2.0 ** -24) * want[fine].abs() * (1 + 2.0 ** -16)).all()


def test_a_workspace_of_more_than_64_gib(L):
    """More than a million tokens of 64 heads behind a prefix: partial results lie further from each other than 2^32 steps of 16 bytes."""
    import torch
    if torch.cuda.mem_get_info()[0] < 125 << 30:
        pytest.skip("needs 125 GB of device memory")
    n_seq, heads, hs, page, prefix = 1_040_000, 64, 128, 8, 8
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v = (torch.randn((2, 1, page, hs), generator=g, device="cuda").bfloat16() for _ in "kv")
    q = torch.empty((n_seq, heads * hs), device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    out = torch.full_like(q, 7.0)
    lengths, table, first = (torch.full(s, x, dtype=torch.int32, device="cuda") for s, x in (((n_seq,), 3), ((n_seq, 1), 1), ((1,), 0)))
    cache = L.PagedCache(dev_k=at(k), dev_v=at(v), type=GGML["bf16"], n_pages=2, page_size=page, n_kv_heads=1, head_size=hs)
    batch = L.PagedBatch(n_seq=n_seq, n_query=1, dev_lengths=at(lengths), dev_pages=at(table), pages_per_seq=1, prefix_len=prefix, dev_prefix_pages=at(first))
    qs = L.PagedQueries(type=GGML["bf16"], n_heads=heads, dev_q=at(q), q_stride=heads * hs, dev_out=at(out), out_stride=heads * hs)
    need = C.c_int64()
    L.check(L.lib().l2b_paged_attention_workspace(C.byref(cache), C.byref(batch), C.byref(qs), C.byref(need)))
    assert need.value > 65 << 30
    w = torch.empty((need.value // 4,), device="cuda")
    L.check(L.lib().l2b_paged_attention_device(C.byref(cache), C.byref(batch), C.byref(qs), at(w), need.value, stream()))
    keys, values = (torch.cat([x[0, 0], x[1, 0, :3]]).double() for x in (k, v))
    rows = torch.cat([torch.arange(0, n_seq, 4999, device="cuda"), torch.arange(n_seq - 40, n_seq, device="cuda")])
    z = torch.softmax(q[rows].double().view(-1, heads, hs) @ keys.T * hs ** -0.5, -1)
    want, size = z @ values, z @ values.abs()
    err = (out[rows].double().view(-1, heads, hs) - want).abs()
    # scores of about 11 in absolute size, off by 2^-18 of it; everything else is smaller
    tol = 2.0 ** -14 * size + 2.0 ** -8 * want.abs()
    bad = ((err > tol).any(-1).any(-1)).nonzero()
    del q, out, w  # (and back to the device: later tests allocate without torch)
    torch.cuda.empty_cache()
    assert len(bad) == 0, (len(bad), rows[bad[0]])


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("n_query,counts,lengths,prefix", [(300, [300, 257, 1], [300, 1000, 40], 0), (701, [701, 0], [1402, 9], 333)])
def test_attention_of_prompts(L, io, cache, n_query, counts, lengths, prefix):
    """Hundreds of new tokens a sequence, with and without positions before them."""
    from test_gpu_paged import check_attention
    b = Batch(L, lengths, n_query=n_query, counts=counts, kv=2, hs=64, page=16, prefix=prefix, cache=cache, seed=n_query)
    check_attention(b, queries(b, 4, io), 4)
