// Attention of a batch's new tokens over a paged cache: softmax(scale * q K^T) V over the positions of a prefix that all sequences share and over the
// sequence's own positions up to the token's.
//
// Rows: the query heads of one key/value head, of all new tokens of a group (a sequence, or all of them for the prefix), in tiles of 16: the M of
// m16n8k16.  What a step of single tokens reads is the cache, once, so memory bounds it; the work is cut into equal shares of 64-key tiles over all
// blocks whatever the sequences' lengths (paged.h), and the partial results (f32 sums, each row's maximum and total) are joined by a second kernel.
// A block is four warps, each with 16 keys of a tile, its own ring of asynchronous 16-byte copies and its own running maximum, total and sums: the
// warps meet at an item's end only.  Copies run ahead over the ends of items.  Rows of keys and values lie 16 bytes further apart in shared memory than
// they are long, so that ldmatrix reads eight rows without bank conflicts.
//
// f32 rows over a 16-bit cache: a query and a weight are split into terms of the cache's type (three of bf16, two of f16, the query's behind a power of two
// per row), which keeps the products' error at 2^-22 or less.  For 16-bit rows the weights are rounded once to the cache's type (at most
// half a step of 2^-8 or 2^-11 relative, as the result itself is); scores, maxima, totals and sums are f32.
#pragma once
#include <type_traits>

#include "paged_append.cuh"

namespace l2b {

constexpr int PT_WARPS = 4, PT_WKEYS = PT_KEYS / PT_WARPS, PT_STAGES = 3;

struct PagedAttnParams : PagedWork {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int n_heads;
    float scale2;          // scale * log2(e)
    int blocks;            // of the own parts' kernel
    float *slot_acc, *slot_ml;  // [2 * blocks][16][hs], [2 * blocks][16][2]
    float *own_acc, *own_ml;    // items that one block did: [rows * n_heads][hs], [..][2]; null where nothing else is to be joined
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
    static constexpr int HALF_STAGE = PT_WKEYS * PITCH;      // keys of a stage, or values
    static constexpr int RING = PT_WARPS * PT_STAGES * 2 * HALF_STAGE;
};
// shared memory: the rings, then each warp's sums, maxima and totals of up to 16 rows
template <typename TR>
__host__ __device__ constexpr int thin_smem(int hs, int rows) { return TR::RING + PT_WARPS * rows * (hs + 2) * 4; }

template <typename T, typename TIO, int KS>
__global__ void __launch_bounds__(PT_WARPS * 32, 2) paged_attention_kernel(const __grid_constant__ PagedAttnParams p) {
    using TR = ThinTraits<T, TIO, KS>;
    extern __shared__ __align__(16) uint8_t pt_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hs = p.pool.hs, chunks = hs / 8, groups = p.seqs.n_seq + p.thin_prefix;
    uint8_t* const ring = pt_smem + warp * PT_STAGES * 2 * TR::HALF_STAGE;
    const int most_rows = min(PT_ROWS, p.seqs.n_query * p.group * (p.thin_prefix ? p.seqs.n_seq : 1));
    float* const merge = reinterpret_cast<float*>(pt_smem + TR::RING);
    // the values between a head's end and the next multiple of 32: zero once and for all
    for (int i = lane; i < PT_STAGES * 2 * PT_WKEYS * (KS * 2 - chunks); i += 32) {
        const int r = i / (KS * 2 - chunks), ch = chunks + i % (KS * 2 - chunks);
        *reinterpret_cast<uint4*>(ring + r * TR::PITCH + ch * 16) = make_uint4(0, 0, 0, 0);
    }
    // The prefix's kernel in front has waited for what was before it, and nothing here hangs on it: then the wait is for the end, so that the joining
    // kernel finds both done.
    const bool late = p.cut.units > 0;
    if (!late) pdl_wait();
    pdl_launch_dependents();  // (behind a wait, here or there: the joining kernel reads the lengths before it waits itself)

    // this block's share; every warp finds it for itself
    int64_t units = 0;
    for (int g = lane; g < groups; g += 32) units += group_units(p, group_shape(p, g));
    for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
    const PagedShares sh = paged_shares(units, p.blocks);
    const int64_t begin = (int64_t)blockIdx.x * sh.share;
    Cursor at;
    at.left = 0;
    if (begin < units) {
        int64_t sum = 0;  // units of the groups before
        int found = -1;
        for (int g0 = 0; found < 0 && g0 < groups; g0 += 32) {
            const int64_t n = g0 + lane < groups ? group_units(p, group_shape(p, g0 + lane)) : 0;
            int64_t inc = n;
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, sum + inc > begin);
            if (hit) {
                const int l = __ffs(hit) - 1;
                sum += __shfl_sync(0xffffffffu, inc - n, l);
                found = g0 + l;
            } else {
                sum += __shfl_sync(0xffffffffu, inc, 31);
            }
        }
        if (found >= 0) at = cursor_at(p, found, begin - sum, min(sh.share, units - begin));
    }

    Cursor ahead = at;
    uint64_t seen = 0;  // 16 bits per stage under way: which of its keys are there
    int in_flight = 0, put_stage = 0, get_stage = 0;
    auto load = [&]() {  // the next tile's 16 keys and values of this warp, or an empty group of copies
        if (ahead.left > 0) {
            const bool pre = p.thin_prefix && ahead.g == 0;
            const int kv = ahead.item / ahead.s.row_tiles, key = ahead.tile * PT_KEYS + warp * PT_WKEYS + (lane & 15);
            int page = -1;
            if (key < ahead.s.keys)
                page = pre ? p.seqs.prefix_pages[key >> p.pool.page_shift] : p.seqs.pages[(int64_t)(ahead.g - p.thin_prefix) * p.seqs.width + (key >> p.pool.page_shift)];
            const bool there = page >= 0 && page < p.pool.n_pages;
            seen |= (uint64_t)(__ballot_sync(0xffffffffu, there) & 0xffffu) << (16 * in_flight);
            const int64_t off = there ? paged_offset(page, kv, key & ((1 << p.pool.page_shift) - 1), p.pool) : 0;
            uint8_t* const st = ring + put_stage * 2 * TR::HALF_STAGE;
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
            next_tile(p, ahead);
        }
        cp_async_commit();
        ++in_flight;
        put_stage = put_stage + 1 == PT_STAGES ? 0 : put_stage + 1;
    };
#pragma unroll 1
    for (int i = 0; i < PT_STAGES - 1; ++i) load();

    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    while (at.left > 0) {
        // one item, or as much of it as is this block's
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
                if (r0 + 8 * i < n_rows) {
                    const int seq = seq0 + t / p.seqs.n_query, j = t % p.seqs.n_query, length = p.seqs.lengths[seq];
                    const int count = paged_count(length, p.seqs.counts ? p.seqs.counts[seq] : p.seqs.n_query, p.seqs.n_query);
                    if (j < count) low[i] = lim[i] = pre ? p.seqs.prefix_len - 1 : length - count + j;
                }
                const TIO* const src = (const TIO*)p.q + token[i] * p.q_stride + (int64_t)head[i] * hs;
                const bool any = lim[i] >= 0;  // (a row without keys here: zeros do)
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
            const int k0 = tile * PT_KEYS + warp * PT_WKEYS;
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
            const bool cut = there != 0xffffu || k0 + PT_WKEYS - 1 > least;
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
            if (k0 + PT_WKEYS - 1 > least) {
                for (int i = lane; i < PT_WKEYS * KS * 2 && !odd; i += 32) {
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
                for (int key = 0; key < PT_WKEYS; ++key) {
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

        // the warps' results together
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (l[i] != l[i] && m[i] == -INFINITY) m[i] = 0.f;  // scores that are no numbers are not an empty row
        }
        __syncthreads();  // (the last item's have been read)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i;
            if (r < most_rows) {
                float* const row = merge + (warp * most_rows + r) * (hs + 2);
#pragma unroll
                for (int n = 0; n < KS * 2; ++n)
                    if (n * 8 < hs) {
                        row[n * 8 + c0] = acc[n][2 * i];
                        row[n * 8 + c0 + 1] = acc[n][2 * i + 1];
                    }
                if ((lane & 3) == 0) {
                    row[hs] = m[i];
                    row[hs + 1] = l[i];
                }
            }
        }
        __syncthreads();
        const bool whole = first_tile == 0 && ends;
        const int slot = 2 * (int)blockIdx.x + (first_tile == 0 ? 1 : 0);
        float* const whole_acc = pre ? p.pre_acc : p.own_acc;
        float* const whole_ml = pre ? p.pre_ml : p.own_ml;
        for (int i = threadIdx.x; i < n_rows * chunks * 2; i += PT_WARPS * 32) {  // four values each
            const int r = i / (chunks * 2), d = (i - r * chunks * 2) * 4;
            float mw[PT_WARPS], top = -INFINITY, sum = 0.f, o[4] = {};
#pragma unroll
            for (int w = 0; w < PT_WARPS; ++w) {
                mw[w] = merge[(w * most_rows + r) * (hs + 2) + hs];
                top = fmaxf(top, mw[w]);
            }
#pragma unroll
            for (int w = 0; w < PT_WARPS; ++w) {
                const float* const row = merge + (w * most_rows + r) * (hs + 2);
                const float f = mw[w] == -INFINITY ? 0.f : exp2_approx(mw[w] - top);
                sum = fmaf(f, row[hs + 1], sum);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] += mw[w] == -INFINITY ? 0.f : f * row[d + e];
            }
            const int rr = row_tile * PT_ROWS + r, t = rr / p.group;
            const int64_t tok = (int64_t)seq0 * p.seqs.n_query + t;
            const int h = kv * p.group + rr - t * p.group;
            if (whole && !whole_acc) {  // all there is of these rows
                const int length = p.seqs.lengths[seq0];
                if (t < paged_count(length, p.seqs.counts ? p.seqs.counts[seq0] : p.seqs.n_query, p.seqs.n_query)) {
                    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] *= inv;
                    put((TIO*)p.out + tok * p.out_stride + (int64_t)h * hs + d, o);
                }
            } else {
                const int64_t at_row = whole ? tok * p.n_heads + h : (int64_t)slot * PT_ROWS + r;
                *reinterpret_cast<float4*>((whole ? whole_acc : p.slot_acc) + at_row * hs + d) = make_float4(o[0], o[1], o[2], o[3]);
                if (d == 0) *reinterpret_cast<float2*>((whole ? whole_ml : p.slot_ml) + at_row * 2) = make_float2(top, sum);
            }
        }
        next_item(p, at, tiles);
    }
    if (late) pdl_wait();
}

// Joins the partial results of a row: a block per token and `heads` heads, a warp's lanes along the head's values.  WARPS warps share a row's parts
// where there are few rows and so many parts of each.
struct JoinParams {
    PagedAttnParams a;
    int heads;  // of a block
};
constexpr int PJ_WARPS = 8;

struct Joined {
    float m, l, o[4];
};
__device__ __forceinline__ void join(Joined& j, float m, float l, const float* acc, bool read) {
    if (m == -INFINITY) return;
    const float mn = fmaxf(j.m, m), a = j.m == -INFINITY ? 0.f : exp2_approx(j.m - mn), b = exp2_approx(m - mn);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (read) v = __ldcg(reinterpret_cast<const float4*>(acc));
    j.l = j.l * a + l * b;
    j.o[0] = j.o[0] * a + v.x * b;
    j.o[1] = j.o[1] * a + v.y * b;
    j.o[2] = j.o[2] * a + v.z * b;
    j.o[3] = j.o[3] * a + v.w * b;
    j.m = mn;
}

template <typename TIO>
__global__ void __launch_bounds__(PJ_WARPS * 32) paged_join_kernel(const __grid_constant__ JoinParams jp) {
    const PagedAttnParams& p = jp.a;
    __shared__ int64_t s_units[2][PJ_WARPS];
    __shared__ float s_part[PJ_WARPS][PA_MAX_SIZE + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hs = p.pool.hs;
    const int64_t tok = blockIdx.x;
    const int seq = (int)(tok / p.seqs.n_query), j = (int)(tok % p.seqs.n_query), group = seq + p.thin_prefix;
    const int length = p.seqs.lengths[seq], count = paged_count(length, p.seqs.counts ? p.seqs.counts[seq] : p.seqs.n_query, p.seqs.n_query);
    // where the shares lie: units of all groups, and of those before this one
    int64_t all = 0, before = 0;
    for (int g = threadIdx.x; g < p.seqs.n_seq + p.thin_prefix; g += PJ_WARPS * 32) {
        const int64_t n = group_units(p, group_shape(p, g));
        all += n;
        before += g < group ? n : 0;
    }
    for (int o = 16; o > 0; o >>= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (lane == 0) {
        s_units[0][warp] = all;
        s_units[1][warp] = before;
    }
    __syncthreads();
    all = before = 0;
    for (int w = 0; w < PJ_WARPS; ++w) {
        all += s_units[0][w];
        before += s_units[1][w];
    }
    const PagedShares sh = paged_shares(all, p.blocks);
    pdl_wait();
    if (j >= count) return;

    const int per_row = PJ_WARPS / jp.heads, head = blockIdx.y * jp.heads + warp / per_row, sub = warp % per_row;
    const bool real = head < p.n_heads;
    const int kv = head / p.group, d = lane * 4;
    const int64_t at_row = tok * p.n_heads + head;
    Joined r = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
    bool done = false;
    auto item = [&](int64_t first_unit, const GroupShape& s, int row, const float* whole_acc, const float* whole_ml) {
        if (s.tiles == 0) return;
        const int row_tile = row / PT_ROWS;
        const int64_t begin = first_unit + ((int64_t)kv * s.row_tiles + row_tile) * s.tiles;
        const PagedParts parts = paged_parts(begin, s.tiles, sh.share);
        if (parts.first == parts.last) {
            if (!whole_acc) done = true;  // written already
            else if (sub == 0) {
                const float2 ml = __ldcg(reinterpret_cast<const float2*>(whole_ml + at_row * 2));
                join(r, ml.x, ml.y, whole_acc + at_row * hs + d, d < hs);
            }
            return;
        }
        for (int b = parts.first + sub; b <= parts.last; b += per_row) {
            const int64_t at = (int64_t)paged_slot(parts, b) * PT_ROWS + row % PT_ROWS;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.slot_ml + at * 2));
            join(r, ml.x, ml.y, p.slot_acc + at * hs + d, d < hs);
        }
    };
    if (real) {
        const int g = head - kv * p.group;
        if (p.cut.units > 0) {
            const int row = (int)(tok * p.group) + g, per_item = p.cut.streams_share * 128, row_tile = row / per_item, r128 = row % 128;
            const int i0 = p.cut.streams_share == 2 ? row % per_item / 128 : 0, streams = p.cut.streams_share == 2 ? 1 : 2;
            const PagedParts parts = paged_parts(((int64_t)kv * p.cut.row_tiles + row_tile) * p.cut.tiles, p.cut.tiles, p.cut.share);
            const bool whole = parts.first == parts.last;
            for (int n = sub; n < (parts.last - parts.first + 1) * streams; n += per_row) {
                const int b = parts.first + n / streams, i = i0 + n % streams;
                const int64_t at = whole ? (streams == 2 ? i * p.cut.whole_rows : 0) + at_row : ((int64_t)paged_slot(parts, b) * 2 + i) * 128 + r128;
                const float2 ml = __ldcg(reinterpret_cast<const float2*>((whole ? p.pre_ml : p.cut_ml) + at * 2));
                join(r, ml.x, ml.y, (whole ? p.pre_acc : p.cut_acc) + at * hs + d, d < hs);
            }
        }
        if (p.thin_prefix) item(0, group_shape(p, 0), (int)(tok * p.group) + g, p.pre_acc, p.pre_ml);
        item(before, group_shape(p, group), j * p.group + g, p.own_acc, p.own_ml);
    }
    if (per_row > 1) {
        if (d < hs)
            for (int e = 0; e < 4; ++e) s_part[warp][d + e] = r.o[e];
        if (lane == 0) {
            s_part[warp][hs] = r.m;
            s_part[warp][hs + 1] = r.l;
        }
        __syncthreads();
        if (sub == 0) {
            for (int w = warp + 1; w < warp + per_row; ++w) {
                const float m = s_part[w][hs], l = s_part[w][hs + 1];
                if (m == -INFINITY) continue;
                const float mn = fmaxf(r.m, m), a = r.m == -INFINITY ? 0.f : exp2_approx(r.m - mn), b = exp2_approx(m - mn);
                r.l = r.l * a + l * b;
                for (int e = 0; e < 4; ++e) r.o[e] = r.o[e] * a + (d < hs ? s_part[w][d + e] * b : 0.f);
                r.m = mn;
            }
        }
    }
    if (real && sub == 0 && !done && d < hs) {
        const float inv = r.l > 0.f ? 1.f / r.l : r.l == 0.f ? 0.f : r.l;
        float o[4];
        for (int e = 0; e < 4; ++e) o[e] = r.o[e] * inv;
        put((TIO*)p.out + tok * p.out_stride + (int64_t)head * hs + d, o);
    }
}

}  // namespace l2b
