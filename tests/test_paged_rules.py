"""CPU checks of the paged cache's entry points: what they refuse, and how the attention's work is cut into shares (paged.h, compiled for the host)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama2.jl_b200", "csrc")
A = 1 << 20  # an address on every boundary; nothing reads it


@pytest.fixture(scope="module")
def L(pkg):
    from llama2_jl_b200 import _lib
    return _lib


def good(L):
    """Descriptors that pass every check (the pointers are never followed: the device check comes behind all others)."""
    cache = L.PagedCache(dev_k=A, dev_v=A, type=L.TYPE_BF16, n_pages=4, page_size=16, n_kv_heads=2, head_size=64)
    batch = L.PagedBatch(n_seq=2, n_query=1, dev_lengths=A, dev_counts=None, dev_pages=A, pages_per_seq=2, prefix_len=5, dev_prefix_pages=A)
    rows = L.PagedRows(type=L.TYPE_F32, n_heads=4, dev_q=A, dev_k=A, dev_v=A, q_stride=256, k_stride=128, v_stride=128, dev_q_out=A, q_out_stride=256, dev_q_gain=A, dev_k_gain=None,
                       eps=1e-6, rope_freq_base=10000.0)
    queries = L.PagedQueries(type=L.TYPE_BF16, n_heads=4, dev_q=A, q_stride=256, dev_out=A, out_stride=256, scale=0.0)
    sampling = L.Sampling(type=L.TYPE_F32, n_rows=2, vocab=100, dev_logits=A, stride=100, dev_uniform=A, dev_tokens=A)
    return dict(cache=cache, batch=batch, rows=rows, queries=queries, sampling=sampling)


def calls(L, d):
    """Status of (append, workspace, attention, sample)."""
    lib, need = L.lib(), C.c_int64()
    c, b = C.byref(d["cache"]), C.byref(d["batch"])
    return (lib.l2b_paged_append_device(c, b, C.byref(d["rows"]), None), lib.l2b_paged_attention_workspace(c, b, C.byref(d["queries"]), C.byref(need)),
            lib.l2b_paged_attention_device(c, b, C.byref(d["queries"]), A, 1 << 40, None), lib.l2b_sample_device(C.byref(d["sampling"]), None))


BAD, TYPE = 1, 2
REFUSED = [
    # descriptor, field, value, status, which of the calls
    ("cache", "dev_k", None, BAD, "awt"), ("cache", "dev_v", A + 8, BAD, "awt"), ("cache", "type", 0, TYPE, "awt"), ("cache", "type", 12, TYPE, "awt"), ("cache", "n_pages", 0, BAD, "awt"),
    ("cache", "page_size", 4, BAD, "awt"), ("cache", "page_size", 24, BAD, "awt"), ("cache", "page_size", 2048, BAD, "awt"), ("cache", "page_size", -16, BAD, "awt"),
    ("cache", "n_kv_heads", 0, BAD, "awt"), ("cache", "n_kv_heads", 3, BAD, "wt"), ("cache", "head_size", 0, BAD, "awt"), ("cache", "head_size", 60, BAD, "awt"), ("cache", "head_size", 136, BAD, "awt"),
    ("batch", "n_seq", -1, BAD, "awt"), ("batch", "n_query", 0, BAD, "awt"), ("batch", "dev_lengths", None, BAD, "awt"), ("batch", "dev_pages", None, BAD, "awt"), ("batch", "pages_per_seq", -1, BAD, "awt"),
    ("batch", "pages_per_seq", 1 << 27, BAD, "awt"), ("batch", "prefix_len", -1, BAD, "awt"), ("batch", "prefix_len", 0x7fffffff, BAD, "awt"), ("batch", "dev_prefix_pages", None, BAD, "awt"),
    ("batch", "n_query", 1 << 30, BAD, "awt"), ("batch", "n_query", 1 << 29, BAD, "wt"),
    ("rows", "type", 1, TYPE, "a"), ("rows", "n_heads", 0, BAD, "a"), ("rows", "dev_q", None, BAD, "a"), ("rows", "dev_q_out", None, BAD, "a"), ("rows", "dev_k", None, BAD, "a"), ("rows", "dev_v", None, BAD, "a"),
    ("rows", "q_stride", 255, BAD, "a"), ("rows", "q_stride", 252, BAD, "a"), ("rows", "k_stride", 130, BAD, "a"), ("rows", "v_stride", 0, BAD, "a"), ("rows", "q_out_stride", 260, BAD, "a"),  # (in place)
   
    ("rows", "dev_k", A + 4, BAD, "a"), ("rows", "dev_q_gain", A + 4, BAD, "a"), ("rows", "eps", -1.0, BAD, "a"), ("rows", "eps", float("nan"), BAD, "a"), ("rows", "rope_freq_base", -2.0, BAD, "a"),
    ("rows", "rope_freq_base", float("inf"), BAD, "a"),
    ("queries", "type", 1, TYPE, "wt"), ("queries", "n_heads", 3, BAD, "wt"), ("queries", "n_heads", 0, BAD, "wt"), ("queries", "dev_q", None, BAD, "t"), ("queries", "dev_out", A + 2, BAD, "t"),
    ("queries", "q_stride", 100, BAD, "t"), ("queries", "out_stride", 257, BAD, "t"), ("queries", "scale", float("nan"), BAD, "wt"), ("queries", "scale", float("inf"), BAD, "wt"),
    ("sampling", "type", 12, TYPE, "s"), ("sampling", "n_rows", -1, BAD, "s"), ("sampling", "vocab", 0, BAD, "s"), ("sampling", "vocab", 393217, BAD, "s"), ("sampling", "stride", 99, BAD, "s"),
    ("sampling", "dev_logits", None, BAD, "s"), ("sampling", "dev_logits", A + 2, BAD, "s"), ("sampling", "dev_uniform", None, BAD, "s"), ("sampling", "dev_uniform", A + 4, BAD, "s"),
    ("sampling", "dev_tokens", None, BAD, "s"), ("sampling", "n_rows", 1 << 29, BAD, "s"),
]


@pytest.mark.parametrize("what,field,value,status,which", REFUSED)
def test_refusals(L, what, field, value, status, which):
    """Refused on the host, with a text, before anything of the device is asked for."""
    d = good(L)
    setattr(d[what], field, value)
    got = dict(zip("awts", calls(L, d)))
    for c in which:
        assert got[c] == status, (c, got)
    for c in set("awts") - set(which):
        assert got[c] != status or what in ("cache", "batch") and status == BAD and got[c] == BAD, (c, got)
    assert L.lib().l2b_last_error_string()


def test_null_descriptors(L):
    d, lib, need = good(L), L.lib(), C.c_int64()
    r = {k: C.byref(v) for k, v in d.items()}
    assert lib.l2b_paged_append_device(None, r["batch"], r["rows"], None) == BAD
    assert lib.l2b_paged_append_device(r["cache"], None, r["rows"], None) == BAD
    assert lib.l2b_paged_append_device(r["cache"], r["batch"], None, None) == BAD
    assert lib.l2b_paged_attention_device(r["cache"], r["batch"], None, A, 1 << 40, None) == BAD
    assert lib.l2b_paged_attention_workspace(r["cache"], r["batch"], r["queries"], None) == BAD
    assert lib.l2b_sample_device(None, None) == BAD


def test_host_memory_and_missing_devices_are_refused(L):
    """Descriptors that are in order, over memory that is no device's: an error, never a launch."""
    import torch
    want = BAD if torch.cuda.is_available() else L.ERR_NO_DEVICE
    assert calls(L, good(L)) == (want,) * 4


SIMULATE = r"""
#include "paged.h"
#include <vector>
using namespace l2b;
// Walks every worker's share as the kernel does.  out: blocks that did each unit of (group, item, tile), in that order; returns the number of units, or a
// negative number where a slot is used twice or a part is missing.
extern "C" long long walk(const int* lengths, int n_seq, int n_query, int width, int page_shift, int prefix_len, int thin_prefix, int n_kv, int group, int blocks, int least, int tile_rows, int* out, long long room) {
    PagedWork w;
    w.pool = {nullptr, nullptr, 1, page_shift, n_kv, 64};
    w.seqs = {lengths, nullptr, nullptr, nullptr, n_seq, n_query, width, prefix_len};
    w.group = group;
    w.thin_prefix = thin_prefix;
    w.tile_shift = tile_rows == 8 ? 3 : 4;
    const int groups = n_seq + thin_prefix;
    std::vector<long long> first(groups + 1, 0);
    for (int g = 0; g < groups; ++g) first[g + 1] = first[g] + group_units(w, group_shape(w, g));
    const long long units = first[groups];
    if (units > room) return -1;
    const PagedShares sh = paged_shares(units, blocks, least);
    std::vector<int> slots(2 * blocks, 0);
    for (int b = 0; b < blocks; ++b) {
        const long long begin = b * sh.share;
        if (begin >= units) continue;
        int g = 0;
        while (first[g + 1] <= begin) ++g;
        auto length = [&](int g) { return group_length(w, g); };
        Cursor at = cursor_at(w, g, group_shape(w, g), begin - first[g], units - begin < sh.share ? units - begin : sh.share), tile = at;
        long long done = 0;
        while (at.left > 0) {
            const int tiles = at.s.tiles - at.tile < at.left ? at.s.tiles - at.tile : (int)at.left;
            const long long unit = first[at.g] + (long long)at.item * at.s.tiles + at.tile;
            for (int t = 0; t < tiles; ++t) {
                if (tile.g != at.g || tile.item != at.item || tile.tile != at.tile + t || tile.left <= 0) return -2;  // the copies run ahead over the same tiles
                ++out[unit + t];
                next_item(w, tile, 1, length);
            }
            const PagedParts parts = paged_parts(unit - at.tile, at.s.tiles, sh.share);
            const bool whole = at.tile == 0 && tiles == at.s.tiles;
            if (whole != (parts.first == parts.last) || b < parts.first || b > parts.last) return -3;
            if (!whole) {
                const int slot = 2 * b + (at.tile == 0 ? 1 : 0);
                if (slot != paged_slot(parts, b) || slots[slot]++) return -4;
            }
            done += tiles;
            next_item(w, at, tiles, length);
        }
        if (done != (units - begin < sh.share ? units - begin : sh.share)) return -5;
    }
    return units;
}
extern "C" int place(int length, int count, int n_query, int width, int page_shift, int* keys) {
    *keys = paged_keys(length, width, page_shift);
    return paged_count(length, count, n_query);
}
extern "C" long long offset(int page, int head, int slot, int page_shift, int n_kv, int hs) { return paged_offset(page, head, slot, {nullptr, nullptr, 1 << 30, page_shift, n_kv, hs}); }
"""


@pytest.fixture(scope="module")
def sim(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "sim.cpp").write_text(SIMULATE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "sim.so"), str(d / "sim.cpp")], check=True)
    lib = C.CDLL(str(d / "sim.so"))
    lib.walk.restype = lib.offset.restype = C.c_longlong
    return lib


@pytest.mark.parametrize("blocks", [1, 7, 148, 1184])
def test_every_tile_belongs_to_one_share(sim, blocks):
    rng = np.random.default_rng(blocks)
    for trial in range(60):
        n_seq, n_query, n_kv, group = int(rng.integers(1, 40)), int(rng.integers(1, 6)), int(rng.integers(1, 9)), int(rng.choice([1, 2, 4, 7, 8]))
        shift, width = int(rng.integers(3, 8)), int(rng.integers(0, 40))
        lengths = rng.integers(-2, (width << shift) + 30, n_seq).astype(np.int32)
        lengths[rng.random(n_seq) < 0.3] = rng.choice([-1, 0, 1, 63, 64, 65])
        prefix = int(rng.choice([0, 1, 63, 64, 65, 1000]))
        thin = int(prefix > 0)
        out, least = np.zeros(1 << 22, np.int32), int(rng.choice([1, 2, 4]))
        tile = int(rng.choice([8, 16]))
        units = sim.walk(lengths.ctypes.data_as(C.c_void_p), n_seq, n_query, width, shift, prefix, thin, n_kv, group, blocks, least, tile, out.ctypes.data_as(C.c_void_p), out.size)
        up = lambda a, b: -(-a // b)  # noqa: E731
        want = sum(up(min(max(int(n), 0), width << shift), 16) for n in lengths) * up(n_query * group, tile) * n_kv + thin * up(prefix, 16) * up(n_seq * n_query * group, tile) * n_kv
        assert units == want
        assert (out[:units] == 1).all() and (out[units:] == 0).all()


def test_places_of_rows(sim):
    keys = C.c_int()
    # length, count, n_query, pages -> new tokens, attended positions
    for length, count, n_query, width, want, room in [(5, 2, 4, 1, 2, 5), (5, 9, 4, 1, 4, 5), (-1, 2, 4, 1, 0, 0), (0, 1, 1, 1, 1, 0), (20, 1, 1, 1, 1, 16), (5, -3, 4, 1, 0, 5), (7, 1, 1, 0, 1, 0),
                                                      (0x7fffffff, 1, 1, 1 << 26, 1, 1 << 30)]:
        assert sim.place(length, count, n_query, width, 4, C.byref(keys)) == want and keys.value == room
    assert sim.offset(600000, 7, 15, 4, 8, 128) == ((600000 * 8 + 7) * 16 + 15) * 128 > 1 << 32
