// Attention of a batch's new tokens over a paged cache: softmax(scale * q K^T) V over the positions of a prefix that all sequences share and over the
// sequence's own positions up to the token's.
//
// Rows: the query heads of one key/value head, of all new tokens of a group (a sequence, or all of them for the prefix), in tiles of 16: the M of
// m16n8k16.  What a step of single tokens reads is the cache, once, so memory bounds it; the work is cut into equal shares of 16-key tiles over all
// warps whatever the sequences' lengths (paged.h), and the partial results (f32 sums, each row's maximum and total) are joined by a second kernel.
// Every warp works by itself: its own share, its own ring of asynchronous 16-byte copies, its own running maximum, total and sums; there is no barrier.  Copies run
// ahead over the ends of items; the page of a tile's keys is looked up one tile before it is needed, and the lengths of 32 sequences at a time.  Rows
// of keys and values lie 16 bytes further apart in shared memory than they are long, so that ldmatrix reads eight rows without bank conflicts.
//
// f32 rows over a 16-bit cache: a query and a weight are split into terms of the cache's type (three of bf16, two of f16, the query's behind a power of two
// per row), which keeps the products' error at 2^-22 or less.  For 16-bit rows the weights are rounded once to the cache's type (at most
// half a step of 2^-8 or 2^-11 relative, as the result itself is); scores, maxima, totals and sums are f32.
#pragma once
#include <type_traits>

#include "paged_append.cuh"

namespace l2b {

constexpr int PT_WARPS = 4, PT_STAGES = 3, PT_LEAST = 2;

struct PagedAttnParams : PagedWork {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int n_heads;
    float scale2;          // scale * log2(e)
    int64_t* starts;            // [groups + 1]: first unit of each group, left by the own parts' kernel for the joining one
    int workers;                // warps of the own parts' kernel
    int slot_rows;              // rows of a slot: 16, or fewer when no tile has as many
    float *slot_acc, *slot_ml;  // [2 * workers][slot_rows][hs], [..][2]
    float *own_acc, *own_ml;    // items that one warp did: [rows * n_heads][hs], [..][2]; null where nothing else is to be joined
    float *pre_acc, *pre_ml;    // the same of the prefix
    PrefixCut cut;              // of the prefix's kernel (paged_prefix.cuh), which may be running still
    float *cut_acc, *cut_ml;    // its slots: [2 * blocks][2][128][hs], [..][2]
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool real) {  // not real: zeros, and nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {  // 2^-22 relative; exp2(-inf) = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two values as a pair of T, and what that leaves of them.
template <typename T>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
    const Pack<T, 2> v = {{from_f32<T>(a), from_f32<T>(b)}};
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ uint32_t split_pair(float& a, float& b) {
    const T x = from_f32<T>(a), y = from_f32<T>(b);
    const Pack<T, 2> v = {{x, y}};
    a -= to_f32(x);
    b -= to_f32(y);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, typename TIO, int KS>
struct ThinTraits {
    static constexpr bool WIDE = sizeof(TIO) == 4;
    static constexpr int QT = !WIDE ? 1 : sizeof(T) == 2 && std::is_same<T, __half>::value ? 2 : 3, PT = QT;
    static constexpr int PITCH = KS * 32 + 16;               // bytes of a row in shared memory
    static constexpr int HALF_STAGE = PT_KEYS * PITCH;      // keys of a stage, or values
    static constexpr int RING = PT_WARPS * PT_STAGES * 2 * HALF_STAGE;
};
// The sequences' lengths as a warp needs them one after the other: 32 at a time.
struct Lengths {
    int base, mine;
    __device__ __forceinline__ int operator()(const PagedWork& p, int g) {
        if (g < base || g >= base + 32) {
            const int lane = threadIdx.x & 31;
            base = g;
            mine = g + lane < p.seqs.n_seq + p.thin_prefix ? group_length(p, g + lane) : 0;
        }
        return __shfl_sync(0xffffffffu, mine, g - base);
    }
};

template <typename T, typename TIO, int KS>
__global__ void __launch_bounds__(PT_WARPS * 32, 2) paged_attention_kernel(const __grid_constant__ PagedAttnParams p) {
    using TR = ThinTraits<T, TIO, KS>;
    extern __shared__ __align__(16) uint8_t pt_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hs = p.pool.hs, chunks = hs / 8, groups = p.seqs.n_seq + p.thin_prefix;
    const int worker = warp * (int)gridDim.x + (int)blockIdx.x;  // (few shares: spread over the SMs)
    uint8_t* const ring = pt_smem + warp * PT_STAGES * 2 * TR::HALF_STAGE;
    // the values between a head's end and the next multiple of 32: zero once and for all
    for (int i = lane; i < PT_STAGES * 2 * PT_KEYS * (KS * 2 - chunks); i += 32) {
        const int r = i / (KS * 2 - chunks), ch = chunks + i % (KS * 2 - chunks);
        *reinterpret_cast<uint4*>(ring + r * TR::PITCH + ch * 16) = make_uint4(0, 0, 0, 0);
    }
    // The prefix's kernel in front has waited for what was before it, and nothing here hangs on it: then the wait is for the end, so that the joining
    // kernel finds both done.
    const bool late = p.cut.units > 0;
    if (!late) pdl_wait();
    pdl_launch_dependents();  // (behind a wait, here or there: the joining kernel reads the lengths before it waits itself)

    // this warp's share
    int64_t units = 0;
    for (int g = lane; g < groups; g += 32) units += group_units(p, group_shape(p, g));
    for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
    const PagedShares sh = paged_shares(units, p.workers, PT_LEAST);
    const int64_t begin = worker * sh.share;
    Cursor at;
    at.left = 0;
    if (begin < units || worker == 0) {
        int64_t sum = 0;  // units of the groups before
        int found = -1;
        if (worker == 0 && lane == 0) p.starts[groups] = units;
        for (int g0 = 0; (found < 0 || worker == 0) && g0 < groups; g0 += 32) {
            const int64_t n = g0 + lane < groups ? group_units(p, group_shape(p, g0 + lane)) : 0;
            int64_t inc = n;
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, sum + inc > begin);
            if (hit && found < 0) {
                const int l = __ffs(hit) - 1;
                found = g0 + l;
                at = cursor_at(p, found, group_shape(p, found), begin - sum - __shfl_sync(0xffffffffu, inc - n, l), min(sh.share, units - begin));
            }
            if (worker == 0 && g0 + lane < groups) p.starts[g0 + lane] = sum + inc - n;
            sum += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    Lengths ahead_lengths = {-64, 0}, at_lengths = {-64, 0};

    Cursor ahead = at;
    uint64_t seen = 0;  // 16 bits per stage under way: which of its keys are there
    int in_flight = 0, put_stage = 0, get_stage = 0;
    int page = -1;  // of this lane's key of the tile that is copied next
    auto look_up = [&]() {
        const int key = ahead.tile * PT_KEYS + (lane & 15);
        page = -1;
        if (ahead.left > 0 && key < ahead.s.keys)
            page = p.thin_prefix && ahead.g == 0 ? p.seqs.prefix_pages[key >> p.pool.page_shift] : p.seqs.pages[(int64_t)(ahead.g - p.thin_prefix) * p.seqs.width + (key >> p.pool.page_shift)];
    };
    look_up();
    auto load = [&]() {  // the next tile's 16 keys and values, or an empty group of copies
        if (ahead.left > 0) {
            const int kv = ahead.item / ahead.s.row_tiles, key = ahead.tile * PT_KEYS + (lane & 15);
            const bool there = page >= 0 && page < p.pool.n_pages;
            seen |= (uint64_t)(__ballot_sync(0xffffffffu, there) & 0xffffu) << (16 * in_flight);
            const int64_t off = there ? paged_offset(page, kv, key & ((1 << p.pool.page_shift) - 1), p.pool) : 0;
            uint8_t* const st = ring + put_stage * 2 * TR::HALF_STAGE;
            next_item(p, ahead, 1, [&](int g) { return ahead_lengths(p, g); });
            look_up();
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const int r = (i * 32 + lane) / (KS * 2), ch = (i * 32 + lane) % (KS * 2);
                const int64_t o = __shfl_sync(0xffffffffu, off, r);
                const bool real = __shfl_sync(0xffffffffu, (int)there, r);
                if (ch < chunks) {
                    cp_async16(st + r * TR::PITCH + ch * 16, (const T*)p.pool.k + o + ch * 8, real);
                    cp_async16(st + TR::HALF_STAGE + r * TR::PITCH + ch * 16, (const T*)p.pool.v + o + ch * 8, real);
                }
            }
        }
        cp_async_commit();
        ++in_flight;
        put_stage = put_stage + 1 == PT_STAGES ? 0 : put_stage + 1;
    };
#pragma unroll 1
    for (int i = 0; i < PT_STAGES - 1; ++i) load();

    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    while (at.left > 0) {
        // one item, or as much of it as is this warp's
        const bool pre = p.thin_prefix && at.g == 0;
        const int kv = at.item / at.s.row_tiles, row_tile = at.item - kv * at.s.row_tiles, first_tile = at.tile;
        const int tiles = (int)min((int64_t)(at.s.tiles - at.tile), at.left);
        const bool ends = at.tile + tiles == at.s.tiles;
        const int seq0 = pre ? 0 : at.g - p.thin_prefix, n_rows = min(PT_ROWS, (pre ? p.seqs.n_seq : 1) * p.seqs.n_query * p.group - row_tile * PT_ROWS);
        // token row and head of this thread's two rows (r0, r0 + 8), and the last key that each sees
        int lim[2], low[2];  // (low: nothing to watch for in rows that are no tokens)
        int64_t token[2];
        int head[2];
        float unscale[2] = {1.f, 1.f};
        uint32_t qa[TR::QT][KS][4];
        {
            float qv[2][KS][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = row_tile * PT_ROWS + r0 + 8 * i, t = r / p.group;
                token[i] = (int64_t)seq0 * p.seqs.n_query + t;
                head[i] = kv * p.group + r - t * p.group;
                lim[i] = -1;
                low[i] = 0x7fffffff;
                const bool any = r0 + 8 * i < n_rows;  // (other rows: zeros do)
                const int seq = any ? seq0 + t / p.seqs.n_query : 0, j = t % p.seqs.n_query, length = p.seqs.lengths[seq], given = p.seqs.counts ? p.seqs.counts[seq] : p.seqs.n_query;
                const TIO* const src = (const TIO*)p.q + token[i] * p.q_stride + (int64_t)head[i] * hs;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int d = ks * 16 + h * 8 + c0;
                        float x[2] = {0.f, 0.f};
                        if (any && d < hs) get(src + d, x);
                        qv[i][ks][2 * h] = x[0];
                        qv[i][ks][2 * h + 1] = x[1];
                    }
                }
                const int count = paged_count(length, given, p.seqs.n_query);
                if (any && j < count) low[i] = lim[i] = pre ? p.seqs.prefix_len - 1 : length - count + j;
                if (TR::WIDE && std::is_same<T, __half>::value) {  // f16 terms: the row's largest value between 1/2 and 1
                    float mx = 0.f;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int h = 0; h < 4; ++h) mx = fmaxf(mx, fabsf(qv[i][ks][h]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    int e = 0;
                    if (mx > 0.f && mx < INFINITY) frexpf(mx, &e);
                    e = max(-100, min(100, e));
                    unscale[i] = ldexpf(1.f, e);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int h = 0; h < 4; ++h) qv[i][ks][h] = ldexpf(qv[i][ks][h], -e);
                }
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int t = 0; t < TR::QT; ++t)
#pragma unroll
                    for (int a = 0; a < 4; ++a) qa[t][ks][a] = split_pair<T>(qv[a & 1][ks][a & 2], qv[a & 1][ks][(a & 2) + 1]);
        }
        int most = max(lim[0], lim[1]), least = min(low[0], low[1]);
        for (int o = 4; o < 32; o <<= 1) {
            most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
        }
        const float sc[2] = {p.scale2 * unscale[0], p.scale2 * unscale[1]};

        float acc[KS * 2][4];
#pragma unroll
        for (int n = 0; n < KS * 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll 1
        for (int tile = first_tile; tile < first_tile + tiles; ++tile) {
            load();
            cp_async_wait<PT_STAGES - 1>();
            __syncwarp();
            const unsigned there = (unsigned)(seen & 0xffffu);
            seen >>= 16;
            --in_flight;
            const uint8_t* const sk = ring + get_stage * 2 * TR::HALF_STAGE;
            const uint8_t* const sv = sk + TR::HALF_STAGE;
            get_stage = get_stage + 1 == PT_STAGES ? 0 : get_stage + 1;
            const int k0 = tile * PT_KEYS;
            if (k0 > most || !there) {  // nobody sees any of it
                __syncwarp();
                continue;
            }
            float s[2][4] = {};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t b[4];  // keys 0-7 and 8-15, the two halves of 16 values each
                ldmatrix4(b, sk + ((lane & 7) + ((lane >> 4) << 3)) * TR::PITCH + (ks * 2 + ((lane >> 3) & 1)) * 16);
#pragma unroll
                for (int t = TR::QT - 1; t >= 0; --t) {
                    mma16<T>(s[0], qa[t][ks], b[0], b[1]);
                    mma16<T>(s[1], qa[t][ks], b[2], b[3]);
                }
            }
            const bool cut = there != 0xffffu || k0 + PT_KEYS - 1 > least;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[n][i] *= sc[i >> 1];
                    const int key = n * 8 + c0 + (i & 1);
                    if (cut && (!(there >> key & 1) || k0 + key > lim[i >> 1])) s[n][i] = -INFINITY;
                }
            float mx[2], use[2], corr[2];
            bool up = false;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                mx[i] = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                up |= mx[i] > m[i];
            }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float mn = fmaxf(m[i], mx[i]);
                    corr[i] = m[i] == -INFINITY ? 0.f : exp2_approx(m[i] - mn);  // (no sums yet)
                    m[i] = mn;
                    l[i] *= corr[i];
                }
#pragma unroll
                for (int n = 0; n < KS * 2; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[n][i] *= corr[i >> 1];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) use[i] = m[i] == -INFINITY ? 0.f : m[i];  // (a row that sees nothing yet)
            float w[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[n][i] = exp2_approx(s[n][i] - use[i >> 1]);
                    l[i >> 1] += w[n][i];
                }
            // A key that one row sees and another does not may hold values that are no numbers: then no product, 0 * inf would spread.
            bool odd = false;
            if (k0 + PT_KEYS - 1 > least) {
                for (int i = lane; i < PT_KEYS * KS * 2 && !odd; i += 32) {
                    const T* v = reinterpret_cast<const T*>(sv + i / (KS * 2) * TR::PITCH + i % (KS * 2) * 16);
                    for (int e = 0; e < 8; ++e) odd |= !(fabsf(to_f32(v[e])) < INFINITY);
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            if (!odd) {
                uint32_t pa[TR::PT][4];
#pragma unroll
                for (int t = 0; t < TR::PT; ++t) {
                    pa[t][0] = split_pair<T>(w[0][0], w[0][1]);
                    pa[t][1] = split_pair<T>(w[0][2], w[0][3]);
                    pa[t][2] = split_pair<T>(w[1][0], w[1][1]);
                    pa[t][3] = split_pair<T>(w[1][2], w[1][3]);
                }
#pragma unroll
                for (int n = 0; n < KS; ++n) {
                    uint32_t b[4];  // values 16n .. 16n+7 and 16n+8 .. 16n+15, the two halves of the keys each
                    ldmatrix4_t(b, sv + ((lane & 7) + (((lane >> 3) & 1) << 3)) * TR::PITCH + (n * 2 + (lane >> 4)) * 16);
#pragma unroll
                    for (int t = TR::PT - 1; t >= 0; --t) {
                        mma16<T>(acc[2 * n], pa[t], b[0], b[1]);
                        mma16<T>(acc[2 * n + 1], pa[t], b[2], b[3]);
                    }
                }
            } else {
                for (int key = 0; key < PT_KEYS; ++key) {
                    const int src = (lane & ~3) | ((key & 7) >> 1);
                    float wk[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float lo = __shfl_sync(0xffffffffu, key < 8 ? w[0][2 * i] : w[1][2 * i], src), hi = __shfl_sync(0xffffffffu, key < 8 ? w[0][2 * i + 1] : w[1][2 * i + 1], src);
                        wk[i] = key & 1 ? hi : lo;
                    }
                    const T* v = reinterpret_cast<const T*>(sv + key * TR::PITCH);
#pragma unroll
                    for (int n = 0; n < KS * 2; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if ((there >> key & 1) && k0 + key <= lim[i >> 1]) acc[n][i] = fmaf(wk[i >> 1], to_f32(v[n * 8 + c0 + (i & 1)]), acc[n][i]);
                }
            }
            __syncwarp();  // the stage may be written again
        }

        // the rows' results: done, or to the workspace
        const bool whole = first_tile == 0 && ends;
        float* const whole_acc = pre ? p.pre_acc : p.own_acc;
        float* const whole_ml = pre ? p.pre_ml : p.own_ml;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i;
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (l[i] != l[i] && m[i] == -INFINITY) m[i] = 0.f;  // scores that are no numbers are not an empty row
            if (r >= n_rows) continue;
            if (whole && !whole_acc) {  // all there is of these rows
                if (low[i] == 0x7fffffff) continue;  // (no token)
                const float inv = l[i] > 0.f ? 1.f / l[i] : l[i] == 0.f ? 0.f : l[i];
                TIO* const dst = (TIO*)p.out + token[i] * p.out_stride + (int64_t)head[i] * hs;
#pragma unroll
                for (int n = 0; n < KS * 2; ++n) {
                    const float o[2] = {acc[n][2 * i] * inv, acc[n][2 * i + 1] * inv};
                    if (n * 8 < hs) put(dst + n * 8 + c0, o);
                }
            } else {
                const int64_t at_row = whole ? token[i] * p.n_heads + head[i] : (int64_t)(2 * worker + (first_tile == 0 ? 1 : 0)) * p.slot_rows + r;
                float* const dst = (whole ? whole_acc : p.slot_acc) + at_row * hs;
#pragma unroll
                for (int n = 0; n < KS * 2; ++n)
                    if (n * 8 < hs) *reinterpret_cast<float2*>(dst + n * 8 + c0) = make_float2(acc[n][2 * i], acc[n][2 * i + 1]);
                if ((lane & 3) == 0) *reinterpret_cast<float2*>((whole ? whole_ml : p.slot_ml) + at_row * 2) = make_float2(m[i], l[i]);
            }
        }
        next_item(p, at, tiles, [&](int g) { return at_lengths(p, g); });
    }
    if (late) pdl_wait();
}

// Joins the partial results of a row (a token's head): a block per token and `heads` heads.  Lanes look up a part each, its maximum and total; then they
// lie along the head's values and add the parts up, so that the loads of many parts are under way at once.  Several warps share a row where there are few.
struct JoinParams {
    PagedAttnParams a;
    int heads;  // of a block
};
constexpr int PJ_WARPS = 8;

template <typename TIO>
__global__ void __launch_bounds__(PJ_WARPS * 32) paged_join_kernel(const __grid_constant__ JoinParams jp) {
    const PagedAttnParams& p = jp.a;
    __shared__ float s_part[PJ_WARPS][PA_MAX_SIZE + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hs = p.pool.hs;
    const int64_t tok = blockIdx.x;
    const int seq = (int)(tok / p.seqs.n_query), j = (int)(tok % p.seqs.n_query), group = seq + p.thin_prefix;
    const int length = p.seqs.lengths[seq], count = paged_count(length, p.seqs.counts ? p.seqs.counts[seq] : p.seqs.n_query, p.seqs.n_query);
    const int per_row = PJ_WARPS / jp.heads, head = blockIdx.y * jp.heads + warp / per_row, sub = warp % per_row;
    const bool real = head < p.n_heads;
    const int kv = head / p.group, g = head - kv * p.group, d = lane * 4;
    const int64_t at_row = tok * p.n_heads + head;

    // the parts of this row: of the prefix's kernel, of the prefix as a group of the own parts' kernel, of the own positions
    const GroupShape own = group_shape(p, group, length), pre = group_shape(p, 0, length);
    const int own_row = j * p.group + g, pre_row = (int)(tok * p.group) + g;
    const int per_item = p.cut.streams_share * 128, streams = p.cut.streams_share == 2 ? 1 : 2;
    PagedParts of[3] = {};
    int n_parts[3] = {};
    if (p.cut.units > 0) {
        of[0] = paged_parts(((int64_t)kv * p.cut.row_tiles + pre_row / per_item) * p.cut.tiles, p.cut.tiles, p.cut.share);
        n_parts[0] = (of[0].last - of[0].first + 1) * streams;
    }
    pdl_wait();
    if (j >= count) return;
    const int64_t units = __ldcg(p.starts + p.seqs.n_seq + p.thin_prefix), share = paged_shares(units, p.workers, PT_LEAST).share;
    if (p.thin_prefix) {
        of[1] = paged_parts(((int64_t)kv * pre.row_tiles + pre_row / PT_ROWS) * pre.tiles, pre.tiles, share);
        n_parts[1] = of[1].last - of[1].first + 1;
    }
    if (own.tiles > 0) {
        of[2] = paged_parts(__ldcg(p.starts + group) + ((int64_t)kv * own.row_tiles + own_row / PT_ROWS) * own.tiles, own.tiles, share);
        n_parts[2] = of[2].last - of[2].first + 1;
    }
    const bool done = own.tiles > 0 && n_parts[2] == 1 && !p.own_acc;  // written already
    const int parts = !real || done ? 0 : n_parts[0] + n_parts[1] + n_parts[2];

    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int first = sub; first < parts; first += 32 * per_row) {  // (the same for the whole warp)
        int n = first + lane * per_row;
        const float *acc = nullptr, *ml = nullptr;
        if (n < parts) {
            if (n < n_parts[0]) {
                const int b = of[0].first + n / streams, i = streams == 1 ? pre_row % per_item / 128 : n % streams;
                const bool whole = of[0].first == of[0].last;
                const int64_t at = whole ? (streams == 2 ? i * p.cut.whole_rows : 0) + at_row : ((int64_t)paged_slot(of[0], b) * 2 + i) * 128 + pre_row % 128;
                acc = (whole ? p.pre_acc : p.cut_acc) + at * hs;
                ml = (whole ? p.pre_ml : p.cut_ml) + at * 2;
            } else {
                const bool of_pre = n < n_parts[0] + n_parts[1];
                const PagedParts& q = of[of_pre ? 1 : 2];
                const bool whole = q.first == q.last;
                n -= of_pre ? n_parts[0] : n_parts[0] + n_parts[1];
                const int64_t at = whole ? at_row : (int64_t)paged_slot(q, q.first + n) * p.slot_rows + (of_pre ? pre_row : own_row) % PT_ROWS;
                acc = (whole ? of_pre ? p.pre_acc : p.own_acc : p.slot_acc) + at * hs;
                ml = (whole ? of_pre ? p.pre_ml : p.own_ml : p.slot_ml) + at * 2;
            }
        }
        float2 v = make_float2(-INFINITY, 0.f);
        if (ml) v = __ldcg(reinterpret_cast<const float2*>(ml));
        const float mn = fmaxf(m, warp_max(v.x)), keep = m == -INFINITY ? 0.f : exp2_approx(m - mn), w = v.x == -INFINITY ? 0.f : exp2_approx(v.x - mn);
        l = l * keep + warp_sum(w * v.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= keep;
        m = mn;
        const unsigned some = __ballot_sync(0xffffffffu, v.x != -INFINITY);
        const int last = 32 - __clz(some);
#pragma unroll 4
        for (int i = 0; i < last; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            const float* const a = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)acc, i));
            if ((some >> i & 1) && d < hs) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(a + d));
                o[0] = fmaf(x.x, wi, o[0]);
                o[1] = fmaf(x.y, wi, o[1]);
                o[2] = fmaf(x.z, wi, o[2]);
                o[3] = fmaf(x.w, wi, o[3]);
            }
        }
    }
    if (per_row > 1) {
        if (d < hs)
            for (int e = 0; e < 4; ++e) s_part[warp][d + e] = o[e];
        if (lane == 0) {
            s_part[warp][hs] = m;
            s_part[warp][hs + 1] = l;
        }
        __syncthreads();
        if (sub == 0) {
            for (int w = warp + 1; w < warp + per_row; ++w) {
                const float mw = s_part[w][hs], lw = s_part[w][hs + 1];
                if (mw == -INFINITY) continue;
                const float mn = fmaxf(m, mw), a = m == -INFINITY ? 0.f : exp2_approx(m - mn), b = exp2_approx(mw - mn);
                l = l * a + lw * b;
                for (int e = 0; e < 4; ++e) o[e] = o[e] * a + (d < hs ? s_part[w][d + e] * b : 0.f);
                m = mn;
            }
        }
    }
    if (real && sub == 0 && !done && d < hs) {
        const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
        for (int e = 0; e < 4; ++e) o[e] *= inv;
        put((TIO*)p.out + tok * p.out_stride + (int64_t)head * hs + d, o);
    }
}

}  // namespace l2b
