// Attention of a batch's new tokens over a paged cache: softmax(scale * q K^T) V over the positions of a prefix that all sequences share and over the
// sequence's own positions up to the token's.
//
// Rows: the query heads of one key/value head, of all new tokens of a group (a sequence, or all of them for the prefix), in tiles of 8 or 16.  Keys are the
// M of m16n8k16 and rows its N (S^T = K Q^T, O^T = V^T P^T), so that the few rows of a step of single tokens leave nothing idle: eight of them take half the
// instructions and registers that they would as an M of 16.  P^T comes from S^T by transposing 8 x 8 blocks in registers.
// What such a step reads is the cache, once, so memory bounds it; the work is cut into equal shares of 16-key tiles over all warps whatever the
// sequences' lengths (paged.h), and the partial results (f32 sums, each row's maximum and total) are joined by a second kernel.
// Every warp works by itself: its own share, its own ring of asynchronous 16-byte copies, its own running maximum, total and sums; there is no barrier.  Copies
// run ahead over the ends of items; the page of a tile's keys is looked up one tile before it is needed, and the lengths of 32 sequences at a time.  Rows
// of keys and values lie 16 bytes further apart in shared memory than they are long, so that ldmatrix reads eight rows without bank conflicts.
//
// Measured: 24 sequences of up to 4001 positions, 24 heads of 96 f16 values, nothing shared (496 MB): 98 to 104 us with the join from one run to another, 0.73 to 0.78 of the
// copy rate; one sequence of 501 positions: 7.6 us and 3.8 for the join, chains of look-ups.
//
// f32 rows over a 16-bit cache: a query and a weight are split into terms of the cache's type (three of bf16, two of f16, the query's behind a power of two
// per row), which keeps the products' error at 2^-22 or less.  For 16-bit rows a weight is two terms (bf16: off by 2^-15 at most, f16: by 2^-22): rounded once
// to the cache's type, weights put the results 0.0022 from the definition's (2-norms, bf16) where the rounding of a result itself is 0.0016.  Scores, maxima, totals and
// sums are f32.
#pragma once
#include <type_traits>

#include "paged_append.cuh"

namespace l2b {

constexpr int PT_WARPS = 4, PT_LEAST = 2;

struct PagedAttnParams : PagedWork {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int n_heads;
    float scale2;          // scale * log2(e)
    int64_t* starts;            // [groups + 1]: first unit of each group, left by the own parts' kernel for the joining one
    int workers;                // warps of the own parts' kernel
    int slot_rows;              // rows of a slot: a tile's, or fewer when no tile has as many
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
// The 8 x 8 block of 16-bit values that a warp holds, a row to four threads, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Two values as a pair of T, and what that leaves of them.
template <typename T>
__device__ __forceinline__ uint32_t split_pair(float& a, float& b) {
    const T x = from_f32<T>(a), y = from_f32<T>(b);
    const Pack<T, 2> v = {{x, y}};
    a -= to_f32(x);
    b -= to_f32(y);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// What the exponents of weights are counted from: the maximum, less `up`.  bf16 has f32's range, but f16's terms stop at steps of 2^-24: behind a maximum of 1, weights of
// 2^-20 would keep four bits, and many such keys may be all there is in a result whose largest weight has a value near zero.  With weights up to 2^15 the steps end at
// 2^-39 of the largest.  Behind a prefix the reference may lag: by 2 for f32 rows, which leaves 2^-38; by 2^6 for 16-bit ones, 2^-33 (128 rows behind 16 000 positions: 128 us;
// with a lag of 2^4 135, of 2 149).  Totals and sums carry the factor; a row's partial results say what they are counted from.  (Beyond 2^23 the difference would not be exact.)
__device__ __forceinline__ float weight_reference(float mx, float up) { return fabsf(mx) < 8388608.f ? mx - up : mx; }

// KS: steps of 16 values of a head, NT: tiles of 8 rows
template <typename T, typename TIO, int KS, int NT>
struct ThinTraits {
    static constexpr bool WIDE = sizeof(TIO) == 4;
    static constexpr int QT = !WIDE ? 1 : std::is_same<T, __half>::value ? 2 : 3, PT = WIDE ? QT : 2;  // terms of queries and of weights
    static constexpr int STAGES = NT == 1 ? 2 : 3, BLOCKS = NT == 1 ? 3 : 2;  // 12 warps of 168 registers on an SM, or 8 of 255
    static constexpr float UP = std::is_same<T, __half>::value ? 15.f : 0.f;  // weights up to 2^15 (weight_reference)
    static constexpr int PITCH = KS * 32 + 16;               // bytes of a row in shared memory
    static constexpr int HALF_STAGE = PT_KEYS * PITCH;       // keys of a stage, or values
    static constexpr int RING = PT_WARPS * STAGES * 2 * HALF_STAGE;
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

template <typename T, typename TIO, int KS, int NT>
__global__ void __launch_bounds__(PT_WARPS * 32, (ThinTraits<T, TIO, KS, NT>::BLOCKS)) paged_attention_kernel(const __grid_constant__ PagedAttnParams p) {
    using TR = ThinTraits<T, TIO, KS, NT>;
    extern __shared__ __align__(16) uint8_t pt_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hs = p.pool.hs, chunks = hs / 8, groups = p.seqs.n_seq + p.thin_prefix;
    const int worker = warp * (int)gridDim.x + (int)blockIdx.x;  // (few shares: spread over the SMs)
    uint8_t* const ring = pt_smem + warp * TR::STAGES * 2 * TR::HALF_STAGE;
    // the values between a head's end and the next multiple of 32: zero once and for all
    for (int i = lane; i < TR::STAGES * 2 * PT_KEYS * (KS * 2 - chunks); i += 32) {
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
        put_stage = put_stage + 1 == TR::STAGES ? 0 : put_stage + 1;
    };
#pragma unroll 1
    for (int i = 0; i < TR::STAGES - 1; ++i) load();

    // this thread's query row as an operand: r0; its rows of scores and sums: c0, c0 + 1 (each of every eight)
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    while (at.left > 0) {
        // one item, or as much of it as is this warp's
        const bool pre = p.thin_prefix && at.g == 0;
        const int kv = at.item / at.s.row_tiles, row_tile = at.item - kv * at.s.row_tiles, first_tile = at.tile;
        const int tiles = (int)min((int64_t)(at.s.tiles - at.tile), at.left);
        const bool ends = at.tile + tiles == at.s.tiles;
        const int seq0 = pre ? 0 : at.g - p.thin_prefix, first_row = row_tile * 8 * NT, n_rows = min(8 * NT, (pre ? p.seqs.n_seq : 1) * p.seqs.n_query * p.group - first_row);
        uint32_t qb[TR::QT][NT][KS][2];
        float unscale[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = first_row + r0 + 8 * nt, t = r / p.group;
            const TIO* const src = (const TIO*)p.q + ((int64_t)seq0 * p.seqs.n_query + t) * p.q_stride + (int64_t)(kv * p.group + r - t * p.group) * hs;
            float qv[KS][4];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = ks * 16 + h * 8 + c0;
                    float x[2] = {0.f, 0.f};
                    if (r0 + 8 * nt < n_rows && d < hs) get(src + d, x);
                    qv[ks][2 * h] = x[0];
                    qv[ks][2 * h + 1] = x[1];
                }
            unscale[nt] = 1.f;
            if (TR::WIDE && std::is_same<T, __half>::value) {  // f16 terms: the row's largest value between 2^14 and 2^15, so that the steps of 2^-24 at which they stop are 2^-38 of it
                float mx = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int h = 0; h < 4; ++h) mx = fmaxf(mx, fabsf(qv[ks][h]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                int e = 0;
                if (mx > 0.f && mx < INFINITY) e = max(-100, ilogbf(mx) + 1) - 15;
                unscale[nt] = ldexpf(1.f, e);
                const float f = ldexpf(1.f, -e);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int h = 0; h < 4; ++h) qv[ks][h] *= f;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t2 = 0; t2 < TR::QT; ++t2) qb[t2][nt][ks][h] = split_pair<T>(qv[ks][2 * h], qv[ks][2 * h + 1]);
        }
        // what each of this thread's rows of scores sees last, and the row's scale
        int lim[2 * NT], most = -1, least = 0x7fffffff;
        float sc[2 * NT];
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
            const int rr = c0 + (i & 1) + 8 * (i >> 1);
            sc[i] = p.scale2 * __shfl_sync(0xffffffffu, unscale[i >> 1], (rr & 7) * 4);
            lim[i] = -1;
            if (rr < n_rows) {
                const int t = (first_row + rr) / p.group, seq = seq0 + t / p.seqs.n_query, j = t % p.seqs.n_query, length = p.seqs.lengths[seq];
                const int count = paged_count(length, p.seqs.counts ? p.seqs.counts[seq] : p.seqs.n_query, p.seqs.n_query);
                if (j < count) {  // (rows that are no tokens: nothing to watch for)
                    lim[i] = pre ? p.seqs.prefix_len - 1 : length - count + j;
                    least = min(least, lim[i]);
                }
            }
            most = max(most, lim[i]);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
        }

        float acc[NT][KS][4];  // [values 16 k + r0, + 8][rows c0, c0 + 1]
        float m[2 * NT], l[2 * NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[nt][k][i] = 0.f;
            m[2 * nt] = m[2 * nt + 1] = -INFINITY;
            l[2 * nt] = l[2 * nt + 1] = 0.f;
        }
#pragma unroll 1
        for (int tile = first_tile; tile < first_tile + tiles; ++tile) {
            load();
            cp_async_wait<TR::STAGES - 1>();
            __syncwarp();
            const unsigned there = (unsigned)(seen & 0xffffu);
            seen >>= 16;
            --in_flight;
            const uint8_t* const sk = ring + get_stage * 2 * TR::HALF_STAGE;
            const uint8_t* const sv = sk + TR::HALF_STAGE;
            get_stage = get_stage + 1 == TR::STAGES ? 0 : get_stage + 1;
            const int k0 = tile * PT_KEYS;
            if (k0 > most || !there) {  // nobody sees any of it
                __syncwarp();
                continue;
            }
            float s[NT][4] = {};  // [keys r0, r0 + 8][rows c0, c0 + 1]
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t a[4];
                ldmatrix4(a, sk + (lane & 15) * TR::PITCH + (ks * 2 + (lane >> 4)) * 16);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int t = TR::QT - 1; t >= 0; --t) mma16<T>(s[nt], a, qb[t][nt][ks][0], qb[t][nt][ks][1]);
            }
            const bool cut = there != 0xffffu || k0 + PT_KEYS - 1 > least;
            float mx[2 * NT];
            bool up = false;
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) {
                float &lo = s[i >> 1][i & 1], &hi = s[i >> 1][2 + (i & 1)];
                lo *= sc[i];
                hi *= sc[i];
                if (cut) {
                    if (!(there >> r0 & 1) || k0 + r0 > lim[i]) lo = -INFINITY;
                    if (!(there >> (r0 + 8) & 1) || k0 + r0 + 8 > lim[i]) hi = -INFINITY;
                }
                mx[i] = fmaxf(lo, hi);
            }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1)
#pragma unroll
                for (int i = 0; i < 2 * NT; ++i) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) {
                if (TR::UP != 0.f) mx[i] = weight_reference(mx[i], TR::UP);
                up |= mx[i] > m[i];
            }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int i = 0; i < 2 * NT; ++i) {
                    const float mn = fmaxf(m[i], mx[i]), corr = m[i] == -INFINITY ? 0.f : exp2_approx(m[i] - mn);  // (no sums yet)
                    m[i] = mn;
                    l[i] *= corr;
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        acc[i >> 1][k][i & 1] *= corr;
                        acc[i >> 1][k][2 + (i & 1)] *= corr;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) {
                const float use = m[i] == -INFINITY ? 0.f : m[i];  // (a row that sees nothing yet)
                float &lo = s[i >> 1][i & 1], &hi = s[i >> 1][2 + (i & 1)];
                lo = exp2_approx(lo - use);
                hi = exp2_approx(hi - use);
                l[i] += lo + hi;
            }
            // A key that one row sees and another does not may hold values that are no numbers: then no product, 0 * inf would spread.
            bool odd = false;
            if (k0 + PT_KEYS - 1 > least) {
#pragma unroll 1
                for (int i = lane; i < PT_KEYS * KS * 2 && !odd; i += 32) {
                    const T* v = reinterpret_cast<const T*>(sv + i / (KS * 2) * TR::PITCH + i % (KS * 2) * 16);
                    for (int e = 0; e < 8; ++e) odd |= !(fabsf(to_f32(v[e])) < INFINITY);
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            if (!odd) {
                uint32_t pb[TR::PT][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int t = 0; t < TR::PT; ++t) {
                        pb[t][nt][0] = transposed(split_pair<T>(s[nt][0], s[nt][1]));
                        pb[t][nt][1] = transposed(split_pair<T>(s[nt][2], s[nt][3]));
                    }
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t a[4];
                    ldmatrix4_t(a, sv + ((lane & 7) + ((lane >> 4) << 3)) * TR::PITCH + (k * 2 + ((lane >> 3) & 1)) * 16);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int t = TR::PT - 1; t >= 0; --t) mma16<T>(acc[nt][k], a, pb[t][nt][0], pb[t][nt][1]);
                }
            } else {
#pragma unroll 1
                for (int key = 0; key < PT_KEYS; ++key) {
                    const T* const v = reinterpret_cast<const T*>(sv + key * TR::PITCH);
#pragma unroll
                    for (int i = 0; i < 2 * NT; ++i) {
                        const float w = __shfl_sync(0xffffffffu, key < 8 ? s[i >> 1][i & 1] : s[i >> 1][2 + (i & 1)], (key & 7) * 4 + (lane & 3));
                        if ((there >> key & 1) && k0 + key <= lim[i]) {
#pragma unroll
                            for (int k = 0; k < KS; ++k) {
                                acc[i >> 1][k][i & 1] = fmaf(w, to_f32(v[k * 16 + r0]), acc[i >> 1][k][i & 1]);
                                acc[i >> 1][k][2 + (i & 1)] = fmaf(w, to_f32(v[k * 16 + 8 + r0]), acc[i >> 1][k][2 + (i & 1)]);
                            }
                        }
                    }
                }
            }
            __syncwarp();  // the stage may be written again
        }

        // the rows' results: done, or to the workspace
        const bool whole = first_tile == 0 && ends;
        float* const whole_acc = pre ? p.pre_acc : p.own_acc;
        float* const whole_ml = pre ? p.pre_ml : p.own_ml;
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
            const int rr = c0 + (i & 1) + 8 * (i >> 1), r = first_row + rr, t = r / p.group;
            for (int o = 4; o < 32; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
            if (l[i] != l[i] && m[i] == -INFINITY) m[i] = 0.f;  // scores that are no numbers are not an empty row
            if (rr >= n_rows) continue;
            const int64_t token = (int64_t)seq0 * p.seqs.n_query + t;
            const int head = kv * p.group + r - t * p.group;
            if (whole && !whole_acc) {  // all there is of these rows
                const int length = p.seqs.lengths[seq0];
                if (t >= paged_count(length, p.seqs.counts ? p.seqs.counts[seq0] : p.seqs.n_query, p.seqs.n_query)) continue;  // (no token)
                const float inv = l[i] > 0.f ? 1.f / l[i] : l[i] == 0.f ? 0.f : l[i];
                TIO* const dst = (TIO*)p.out + token * p.out_stride + (int64_t)head * hs + r0;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    if (k * 16 < hs) dst[k * 16] = from_f32<TIO>(acc[i >> 1][k][i & 1] * inv);
                    if (k * 16 + 8 < hs) dst[k * 16 + 8] = from_f32<TIO>(acc[i >> 1][k][2 + (i & 1)] * inv);
                }
            } else {
                const int64_t at_row = whole ? token * p.n_heads + head : (int64_t)(2 * worker + (first_tile == 0 ? 1 : 0)) * p.slot_rows + rr;
                float* const dst = (whole ? whole_acc : p.slot_acc) + at_row * hs + r0;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    if (k * 16 < hs) dst[k * 16] = acc[i >> 1][k][i & 1];
                    if (k * 16 + 8 < hs) dst[k * 16 + 8] = acc[i >> 1][k][2 + (i & 1)];
                }
                if (r0 == 0) *reinterpret_cast<float2*>((whole ? whole_ml : p.slot_ml) + at_row * 2) = make_float2(m[i], l[i]);
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
    int heads;  // of a block: PJ_WARPS, or 1
};
constexpr int PJ_WARPS = 8;

template <typename TIO>
__global__ void __launch_bounds__(PJ_WARPS * 32) paged_join_kernel(const __grid_constant__ JoinParams jp) {
    const PagedAttnParams& p = jp.a;
    __shared__ float s_part[PJ_WARPS][PA_MAX_SIZE + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hs = p.pool.hs;
    const uint32_t tok = blockIdx.x, seq = tok / (uint32_t)p.seqs.n_query, j = tok - seq * (uint32_t)p.seqs.n_query, group = seq + p.thin_prefix;
    const int length = p.seqs.lengths[seq], count = paged_count(length, p.seqs.counts ? p.seqs.counts[seq] : p.seqs.n_query, p.seqs.n_query);
    const int per_row_shift = jp.heads == PJ_WARPS ? 0 : 3, per_row = 1 << per_row_shift, head = blockIdx.y * jp.heads + (warp >> per_row_shift), sub = warp & (per_row - 1);
    const bool real = head < p.n_heads;
    const uint32_t kv = (uint32_t)head / (uint32_t)p.group;
    const int g = head - (int)kv * p.group, d = lane * 4;
    const uint32_t at_row = tok * (uint32_t)p.n_heads + head;

    // the parts of this row: of the prefix's kernel, of the prefix as a group of the own parts' kernel, of the own positions
    const GroupShape own = group_shape(p, group, length), pre = group_shape(p, 0, length);
    const uint32_t own_row = j * p.group + g, pre_row = tok * p.group + g, tile_shift = p.tile_shift, tile_mask = (1u << p.tile_shift) - 1u;
    const int item_shift = p.cut.streams_share == 2 ? 8 : 7, stream_shift = p.cut.streams_share == 2 ? 0 : 1;
    PagedParts of[3] = {};
    int n_parts[3] = {};
    if (p.cut.units > 0) {
        of[0] = paged_parts(((int64_t)kv * p.cut.row_tiles + (pre_row >> item_shift)) * p.cut.tiles, p.cut.tiles, p.cut.share);
        n_parts[0] = (of[0].last - of[0].first + 1) << stream_shift;
    }
    pdl_wait();
    if ((int)j >= count) return;
    const int64_t units = __ldcg(p.starts + p.seqs.n_seq + p.thin_prefix), start = __ldcg(p.starts + group), share = paged_shares(units, p.workers, PT_LEAST).share;
    if (p.thin_prefix) {
        of[1] = paged_parts(((int64_t)kv * pre.row_tiles + (pre_row >> tile_shift)) * pre.tiles, pre.tiles, share);
        n_parts[1] = of[1].last - of[1].first + 1;
    }
    if (own.tiles > 0) {
        of[2] = paged_parts(start + ((int64_t)kv * own.row_tiles + (own_row >> tile_shift)) * own.tiles, own.tiles, share);
        n_parts[2] = of[2].last - of[2].first + 1;
    }
    const bool done = own.tiles > 0 && n_parts[2] == 1 && !p.own_acc;  // written already
    const int parts = !real || done ? 0 : n_parts[0] + n_parts[1] + n_parts[2];

    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int first = sub; first < parts; first += 32 << per_row_shift) {  // (the same for the whole warp)
        int n = first + (lane << per_row_shift);
        const float *acc = nullptr, *ml = nullptr;
        if (n < n_parts[0]) {
            const int b = of[0].first + (n >> stream_shift), i = stream_shift ? n & 1 : (pre_row >> 7) & 1;
            const bool whole = of[0].first == of[0].last;
            const int64_t at = whole ? (stream_shift ? i * p.cut.whole_rows : 0) + at_row : ((int64_t)paged_slot(of[0], b) * 2 + i) * 128 + (pre_row & 127);
            acc = (whole ? p.pre_acc : p.cut_acc) + at * hs;
            ml = (whole ? p.pre_ml : p.cut_ml) + at * 2;
        } else if (n < parts) {
            const bool of_pre = n < n_parts[0] + n_parts[1];
            const PagedParts q = of_pre ? of[1] : of[2];
            const bool whole = q.first == q.last;
            n -= of_pre ? n_parts[0] : n_parts[0] + n_parts[1];
            const int64_t at = whole ? (int64_t)at_row : (int64_t)paged_slot(q, q.first + n) * p.slot_rows + ((of_pre ? pre_row : own_row) & tile_mask);
            acc = (whole ? of_pre ? p.pre_acc : p.own_acc : p.slot_acc) + at * hs;
            ml = (whole ? of_pre ? p.pre_ml : p.own_ml : p.slot_ml) + at * 2;
        }
        float2 v = make_float2(-INFINITY, 0.f);
        if (ml) v = __ldcg(reinterpret_cast<const float2*>(ml));
        const int64_t off = acc ? (acc - p.slot_acc) >> 2 : 0;  // (in steps of 16 bytes; 64 bits: a million tokens' partial results are more than 64 GiB)
        const int last = min(32, (parts - first + per_row - 1) >> per_row_shift);
        // the sums of four parts under way while the maxima come
        auto take = [&](int i, float4& x) {
            const int64_t at = __shfl_sync(0xffffffffu, off, i);
            x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i < last && d < hs) x = __ldcg(reinterpret_cast<const float4*>(p.slot_acc) + at + lane);
        };
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) take(i, x[i]);
        const float mn = fmaxf(m, warp_max(v.x)), keep = m == -INFINITY ? 0.f : exp2_approx(m - mn), w = v.x == -INFINITY ? 0.f : exp2_approx(v.x - mn);
        l = l * keep + warp_sum(w * v.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= keep;
        m = mn;
        const unsigned some = __ballot_sync(0xffffffffu, v.x != -INFINITY);
        for (int i0 = 0; i0 < last; i0 += 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float wi = __shfl_sync(0xffffffffu, w, (i0 + i) & 31);
                if (i0 + i < last && (some >> (i0 + i) & 1)) {
                    o[0] = fmaf(x[i].x, wi, o[0]);
                    o[1] = fmaf(x[i].y, wi, o[1]);
                    o[2] = fmaf(x[i].z, wi, o[2]);
                    o[3] = fmaf(x[i].w, wi, o[3]);
                }
            }
            if (i0 + 4 < last) {
#pragma unroll
                for (int i = 0; i < 4; ++i) take((i0 + 4 + i) & 31, x[i]);
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
        put((TIO*)p.out + (int64_t)tok * p.out_stride + (int64_t)head * hs + d, o);
    }
}

}  // namespace l2b
