"""Filtered sampling on device pointers (l2b_sample_device) against its definition in 64 bits: tokens are equal, probabilities to f32's half step.

The definition's masses are f64 sums; the kernel's are multiples of 2^-44 of the largest weight.  A row whose random number lies within 1e-9 of a border of the
cumulated masses, or whose nucleus or min-p border is that near, could fall either way; the inputs are seeded, and the reference asserts that none does."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
GGML = {"f32": 0, "f16": 1, "bf16": 30}


@pytest.fixture(scope="module")
def L(pkg):
    from llama2_jl_b200 import _lib
    _lib.lib()
    return _lib


def reference(x, t=1.0, k=0, p=1.0, m=0.0, u=0.5, margin=1e-9):
    """(token, probability) of a row of f64 logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return -1, 0.0
    top = int(np.argmax(x))
    if not t > 0:
        return top, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / t))
    w = np.where(x > -np.inf, w, 0.0)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if 0 < k < len(order):
        order = order[:k]
    if p < 1:
        before = np.concatenate(([0.0], np.cumsum(w[order])[:-1]))
        whole = w[order].sum()
        assert margin == 0 or np.abs(before - p * whole)[1:].min(initial=1.0) > margin * whole or p <= 0
        order = order[:max(1, int((before < p * whole).sum()))]
    if m > 0:
        assert margin == 0 or np.abs(w[order] - m)[1:].min(initial=1.0) > 1e-12
        order = order[[i == 0 or w[o] >= m for i, o in enumerate(order)]]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    assert margin == 0 or np.abs(run[:-1] - u * run[-1]).min(initial=1.0) > margin * run[-1]
    at = min(int((run <= u * run[-1]).sum()), len(kept) - 1)
    return int(kept[at]), float(w[kept[at]] / run[-1])


def sample(L, logits, stride=None, vocab=None, probs=True, **settings):
    """logits: a torch tensor [rows, >= vocab]; settings as arrays or numbers for all rows."""
    import torch
    rows, vocab = logits.shape[0], vocab or logits.shape[1]
    kind = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}[logits.dtype]
    types = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32, uniform=torch.float64)
    dev = {n: torch.as_tensor(np.broadcast_to(np.asarray(v), (rows,)).copy()).to("cuda", types[n]) for n, v in settings.items()}
    tokens, got = torch.full((rows + 1,), -9, dtype=torch.int32, device="cuda"), torch.full((rows + 1,), -9.0, device="cuda")
    a = L.Sampling(type=kind, n_rows=rows, vocab=vocab, dev_logits=logits.data_ptr(), stride=logits.stride(0), dev_tokens=tokens.data_ptr(), dev_probs=got.data_ptr() if probs else None,
                   **{"dev_" + n: v.data_ptr() for n, v in dev.items()})
    L.check(L.lib().l2b_sample_device(C.byref(a), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert int(tokens[rows]) == -9 and float(got[rows]) == -9
    return tokens[:rows].tolist(), got[:rows].tolist()


def check(L, logits, margin=1e-9, **s):
    tokens, probs = sample(L, logits, **s)
    x = logits.double().cpu().numpy()
    short = dict(temperature="t", top_k="k", top_p="p", min_p="m", uniform="u")
    for r in range(x.shape[0]):
        one = {short[n]: (float if n == "uniform" else int if n == "top_k" else lambda v: float(np.float32(v)))(np.broadcast_to(np.asarray(v), (x.shape[0],))[r]) for n, v in s.items()}
        token, prob = reference(x[r], margin=margin, **one)
        assert tokens[r] == token, (r, tokens[r], token, one)
        # f32's half step of the quotient, and masses of whole multiples of 2^-44 out of at least 1
        assert abs(probs[r] - prob) <= 2.0 ** -24 * prob + x.shape[1] * 2.0 ** -45, (r, probs[r], prob)


def logits(rows, vocab, seed, io="f32", spread=2.5):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g, device="cuda") * spread).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[io])


def uniforms(rows, seed):
    return np.random.default_rng(seed).random(rows)


CUTS = [dict(), dict(top_k=1), dict(top_k=40), dict(top_k=900), dict(top_k=5000), dict(top_p=0.9), dict(top_p=0.3), dict(top_p=0.999), dict(min_p=0.05), dict(min_p=0.9), dict(top_k=50, top_p=0.8),
        dict(top_k=3000, top_p=0.97), dict(top_k=100, top_p=0.95, min_p=0.02), dict(top_p=0.95, min_p=0.01)]


@pytest.mark.parametrize("cuts", CUTS)
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (6, 32000), (40, 4099), (3, 17), (5, 1), (2, 2), (150, 700)])
def test_cuts(L, rows, vocab, cuts):
    check(L, logits(rows, vocab, vocab + rows), temperature=0.8, uniform=uniforms(rows, vocab), **cuts)


@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cuts", [dict(), dict(top_k=30, top_p=0.9), dict(top_p=0.97), dict(min_p=0.03)])
def test_types_and_strides(L, io, cuts):
    """16-bit logits have many equal values: the lower index comes first.  Rows at odd places."""
    big = logits(9, 5003, 1, io)
    check(L, big[:, 1:4998], temperature=1.1, uniform=uniforms(9, 2), margin=1e-10, **cuts)


def test_settings_row_by_row(L):
    r = np.random.default_rng(4)
    n = 64
    check(L, logits(n, 20011, 3), temperature=np.where(r.random(n) < 0.2, 0.0, r.uniform(0.2, 2.0, n)), top_k=r.choice([0, -3, 1, 7, 200, 30000], n), top_p=r.choice([1.0, 2.0, 0.5, 0.9], n),
          min_p=r.choice([0.0, -1.0, 0.02, 0.3], n), uniform=r.random(n))


@pytest.mark.parametrize("rows", [1, 3, 30, 160, 700])
def test_the_row_alone_decides(L, rows):
    """The same row among others, whatever the number of blocks per row: same token, same probability, twice."""
    import torch
    one = logits(1, 30011, 6)
    for cuts in (dict(), dict(top_k=80), dict(top_p=0.93), dict(top_k=2500, top_p=0.9)):
        s = dict(temperature=0.9, uniform=0.613, **cuts)
        want = sample(L, one, **s)
        many = torch.cat([logits(rows // 2, 30011, 7), one, logits(rows - rows // 2, 30011, 8)])
        for _ in range(2):
            tokens, probs = sample(L, many, **s)
            assert (tokens[rows // 2], probs[rows // 2]) == (want[0][0], want[1][0])


@pytest.mark.parametrize("cuts", [dict(top_k=700), dict(top_p=0.4), dict(top_k=6000, top_p=0.5), dict(min_p=0.5)])
def test_equal_logits(L, cuts):
    """More equal values than a list holds: the lower index first, cut in the middle of them.  Weights are whole multiples of the unit, so the
    borders of these rows are exact."""
    import torch
    x = torch.zeros((4, 9000), device="cuda")
    x[1, 100:] = -0.0
    x[2, ::2] = 3.0
    x[3, 4000] = 1.0
    check(L, x, temperature=1.0, uniform=np.array([0.25, 0.77, 0.5001, 0.9]), margin=0, **cuts)


def test_no_numbers_and_infinities(L):
    import torch
    x = logits(8, 3000, 9)
    x[0, :] = float("nan")
    x[1, :] = -float("inf")
    x[2, :] = -float("inf")
    x[2, 2999] = -1e30
    x[3, 5] = float("nan")
    x[3, 1000:] = -float("inf")
    x[4, 7] = x[4, 70] = x[4, 2999] = float("inf")
    x[5, 0], x[5, 1] = 3e38, -3e38
    x[6, :] = -3e38
    x[7, 100:] = -1e9
    for cuts in (dict(), dict(top_k=2), dict(top_k=50, top_p=0.9), dict(top_p=0.6), dict(min_p=0.1)):
        check(L, x, temperature=0.7, uniform=np.full(8, 0.41), margin=0, **cuts)
    tokens, probs = sample(L, x, temperature=0.0, uniform=0.5)
    assert tokens[0] == tokens[1] == -1 and probs[0] == probs[1] == 0 and tokens[4] == 7


@pytest.mark.parametrize("t", [1e-30, 1e-4, 0.05, 30.0, 1e20, float("inf"), -1.0, float("nan")])
def test_temperatures(L, t):
    for cuts in (dict(), dict(top_k=33), dict(top_p=0.7)):
        check(L, logits(3, 5000, 12), temperature=t, uniform=uniforms(3, 5), margin=1e-10, **cuts)


def test_ends_of_the_random_number(L):
    """0 takes the first kept token, numbers just below 1 the last one with mass; what lies outside is taken as the nearer end."""
    x = logits(1, 4000, 13)
    a = x[0].double().cpu().numpy()
    kept = np.sort(np.argsort(-a, kind="stable")[:25])
    for u, want in ((0.0, kept[0]), (-3.0, kept[0]), (float("nan"), kept[0]), (1 - 2.0 ** -53, kept[-1]), (1.0, kept[-1]), (9.0, kept[-1])):
        assert sample(L, x, temperature=1.0, top_k=25, uniform=u)[0][0] == want, u
    for u, want in ((0.0, 0), (1.0, 3999)):
        assert sample(L, x, temperature=5.0, uniform=u, probs=False)[0][0] == want


def test_no_cuts_given(L):
    check(L, logits(4, 1000, 14), uniform=uniforms(4, 6))


def test_largest_vocabulary(L):
    for cuts in (dict(top_k=60), dict(top_p=0.9)):
        check(L, logits(2, 393216, 15), temperature=0.6, uniform=uniforms(2, 7), margin=1e-10, **cuts)


def test_frequencies(L):
    """Evenly spread random numbers draw every token as often as its probability says: counts are off by at most one border at each end."""
    import torch
    n = 4000
    x = torch.log(torch.tensor([0.1, 0.4, 0.0, 0.3, 0.2], device="cuda"))
    tokens, _ = sample(L, x.repeat(n, 1), uniform=(np.arange(n) + 0.5) / n)
    counts = np.bincount(tokens, minlength=5) / n
    assert np.abs(counts - [0.1, 0.4, 0.0, 0.3, 0.2]).max() <= 2 / n


def test_in_a_graph(L):
    import torch
    x, u = logits(3, 32000, 16), torch.rand(3, dtype=torch.float64, device="cuda")
    tokens, k = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.full((3,), 50, dtype=torch.int32, device="cuda")
    a = L.Sampling(type=0, n_rows=3, vocab=32000, dev_logits=x.data_ptr(), stride=32000, dev_top_k=k.data_ptr(), dev_uniform=u.data_ptr(), dev_tokens=tokens.data_ptr())
    call = lambda: L.check(L.lib().l2b_sample_device(C.byref(a), torch.cuda.current_stream().cuda_stream))  # noqa: E731
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for seed in (17, 18):
        x.copy_(logits(3, 32000, seed))
        u.copy_(torch.rand(3, dtype=torch.float64, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        for r in range(3):
            assert int(tokens[r]) == reference(x[r].double().cpu().numpy(), k=50, u=float(u[r]), margin=0)[0]
    assert math.isfinite(float(u.sum()))
