// Arithmetic of the paged cache that the append and attention kernels and their host side share: which rows of a batch are new tokens, where a
// position lies, and how the attention's work is cut into equal shares.  Plain C++ (the tests compile it for the host too).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define L2B_HD __host__ __device__ __forceinline__
#else
#define L2B_HD inline
#endif

namespace l2b {

// Pages [n_pages][n_kv][page_size][hs] of 16-bit values, for keys and for values.
struct PagedPool {
    void *k, *v;
    int n_pages, page_shift, n_kv, hs;
};
// A batch: sequence i has rows i * n_query .. of which the first count(i) are new tokens.
struct PagedSeqs {
    const int *lengths, *counts, *pages, *prefix_pages;
    int n_seq, n_query, width, prefix_len;
};

// New tokens of a sequence; none of one that sits this step out (a negative length).
L2B_HD int paged_count(int length, int count, int n_query) { return length < 0 || count < 0 ? 0 : count < n_query ? count : n_query; }
// Own positions that a sequence's page table has room for (at most 2^31 - 1: the entry points see to it).
L2B_HD int paged_keys(int length, int width, int page_shift) {
    const int64_t room = (int64_t)width << page_shift;
    return length < 0 ? 0 : length < room ? length : (int)room;
}
L2B_HD int64_t paged_offset(int page, int head, int slot, const PagedPool& p) {
    return ((((int64_t)page * p.n_kv + head) << p.page_shift) + slot) * p.hs;
}

// The attention's work in units of one tile of keys: items (a tile of rows of one key/value head of one group, a group being a sequence or the
// shared prefix) lie one behind the other, each as long as its group has key tiles, and worker c of n (a warp, or a block) takes units c * share ..  An item that
// falls into one share is done there; of a longer one each worker leaves a partial result: the one with which it begins in its second slot, the others
// in their first.  A worker has at most one item of either kind.
struct PagedShares {
    int64_t units, share;
};
L2B_HD PagedShares paged_shares(int64_t units, int workers, int least) {
    PagedShares s;
    s.units = units;
    s.share = units + workers <= 0xffffffffll ? ((uint32_t)units + (uint32_t)workers - 1u) / (uint32_t)workers : (units + workers - 1) / workers;
    if (s.share < least) s.share = least;
    return s;
}
struct PagedParts {
    int first, last;  // workers
};
L2B_HD PagedParts paged_parts(int64_t begin, int tiles, int64_t share) {
    PagedParts p;
    if (begin + tiles <= 0xffffffffll) {  // (a 64-bit division is a hundred instructions; the share is no larger than all units)
        const uint32_t b = (uint32_t)begin, s = share <= 0xffffffffll ? (uint32_t)share : 0xffffffffu;
        p.first = (int)(b / s);
        p.last = (int)((b + (uint32_t)tiles - 1u) / s);
    } else {
        p.first = (int)(begin / share);
        p.last = (int)((begin + tiles - 1) / share);
    }
    return p;
}
L2B_HD int paged_slot(const PagedParts& p, int worker) { return 2 * worker + (worker == p.first ? 1 : 0); }


// How the prefix's kernel cuts its work: row tiles of `streams_share` * 128 rows; streams_share 2: two row tiles on the same keys, 1: one, whose keys
// the two streams take in turn.  units 0: there is no such part.
struct PrefixCut {
    int64_t units, share, whole_rows;  // whole_rows: rows of the batch * heads
    int tiles, row_tiles, streams_share;
};

constexpr int PT_KEYS = 16;  // of a tile of the own parts' kernel

// Rows of a group are the query heads of one key/value head, of all the group's rows one after the other.  Groups: the prefix first where it is one
// (thin_prefix), then the sequences.
struct PagedWork {
    PagedPool pool;
    PagedSeqs seqs;
    int group;  // query heads of a key/value head
    int thin_prefix;
    int tile_shift;  // a tile has 8 rows or 16
};
struct GroupShape {
    int keys, tiles, row_tiles;
};
L2B_HD GroupShape group_shape(const PagedWork& p, int g, int length) {  // length: of the sequence; none of the prefix
    GroupShape s;
    const bool pre = p.thin_prefix && g == 0;
    s.keys = pre ? p.seqs.prefix_len : paged_keys(length, p.seqs.width, p.pool.page_shift);
    s.row_tiles = (int)(((int64_t)(pre ? p.seqs.n_seq : 1) * p.seqs.n_query * p.group + (1 << p.tile_shift) - 1) >> p.tile_shift);
    s.tiles = s.keys / PT_KEYS + (s.keys % PT_KEYS != 0);
    return s;
}
L2B_HD int group_length(const PagedWork& p, int g) { return p.thin_prefix && g == 0 ? 0 : p.seqs.lengths[g - p.thin_prefix]; }
L2B_HD GroupShape group_shape(const PagedWork& p, int g) { return group_shape(p, g, group_length(p, g)); }
L2B_HD int64_t group_units(const PagedWork& p, const GroupShape& s) { return (int64_t)s.tiles * s.row_tiles * p.pool.n_kv; }

// A place in a worker's share: unit `tile` of item `item` (key/value head * row_tiles + row tile) of group `g`.
struct Cursor {
    int g, item, tile;
    GroupShape s;
    int64_t left;  // units of the share from here on
};
L2B_HD Cursor cursor_at(const PagedWork& p, int g, const GroupShape& s, int64_t unit_of_group, int64_t left) {
    Cursor c;
    c.g = g;
    c.s = s;
    if (unit_of_group <= 0xffffffffll) {  // (as above: no 64-bit division where none is needed)
        c.item = (int)((uint32_t)unit_of_group / (uint32_t)s.tiles);
        c.tile = (int)((uint32_t)unit_of_group - (uint32_t)c.item * (uint32_t)s.tiles);
    } else {
        c.item = (int)(unit_of_group / s.tiles);
        c.tile = (int)(unit_of_group % s.tiles);
    }
    c.left = left;
    return c;
}
// `tiles` of the item on, to the next item (of a group that has any) at its end.  length(g): as group_length.
template <class Length>
L2B_HD void next_item(const PagedWork& p, Cursor& c, int tiles, Length&& length) {
    c.left -= tiles;
    c.tile += tiles;
    if (c.tile < c.s.tiles) return;
    c.tile = 0;
    if (++c.item < c.s.row_tiles * p.pool.n_kv) return;
    c.item = 0;
    while (c.left > 0) {
        if (++c.g >= p.seqs.n_seq + p.thin_prefix) c.left = 0;  // (not while the lengths are what they were)
        else if ((c.s = group_shape(p, c.g, length(c.g))).tiles > 0) return;
    }
}

}  // namespace l2b
