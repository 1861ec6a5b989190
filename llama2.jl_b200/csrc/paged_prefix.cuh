// The shared prefix's part of the paged attention on the 5th-generation tensor cores: the rows of all sequences (every query head of a key/value
// head, of every new token) against the same keys, which are read once per 256 (128) rows instead of once per sequence.
//
// A block runs two streams, each with its own 128 rows of scores and sums in tensor memory and its own four softmax warps (a thread per row), so that
// one's products run beside the other's exponentials:  S = Q K^T,  P = exp2(S - m) as a tensor-memory operand in S's place,  O += P V.
//   TILES = 2: the streams are two row tiles that share the tiles of keys (128 each);
//   TILES = 1: one row tile, the streams take the tiles of keys in turn and leave a partial result each: for few rows, and for f32 rows, whose three (f16: two)
//              terms of Q take the place of a second tile (64 keys a tile).
// The scores come in steps of 64 keys.  16-bit rows have two buffers of them, so that the next step's Q K^T is done before this step's exponentials are: with one
// buffer of 128 keys a stream waited 2000 of 3900 cycles per tile for its products (P was one term then: attention behind 16 000 positions took 128 us instead of 116).
//   warps 0-3, 4-7  the streams' softmax; before it they bring the block's rows of Q into shared memory, after it the sums to the workspace
//   warps 8, 10     issue a stream's products each: P V of a step, then Q K^T of the step that gets its buffer
//   warp 9          TMA copies of keys and values straight from the pages: 8 rows or more at a time, V's rows behind the prefix's end through a map
//                   that ends there, so that they are zeros; pages that are none lie outside the map and are zeros, too
// Rows are rescaled only when a maximum has grown by more than 2^8 (f16 caches: 2^6, f32 rows over them: 2), and then all 32 of a warp.  The work, items (key/value
// head, row tile) of the prefix' key tiles, is cut into equal shares of a block per SM (paged.h).  Every wait is bounded; a block whose wait ran out leaves NaN.
// Measured: 128 rows of 64 heads over 8 x 16 000 keys of 128 values (67.1 GFLOP): a call takes 124 us with keys and values in the cache, 132 to 134 with new ones, of which own
// parts 24 and the join 14; what is left, 86 to 94, is 0.71 to 0.78 PFLOP/s.  The tensor pipe, for which P's second term is half as much again, is 63 % active, the
// exponential unit 43 %: bound by a stream's chain scores - maximum - exponentials - terms, whose phases overlap in part.
#pragma once
#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace l2b {

constexpr int PX_ROWS = 128, PX_THREADS = 352, PX_MAX_STAGES = 8, PX_RING = 16;  // PX_RING: masks under way, more than stages

struct PrefixParams : PagedWork {
    const void* q;
    int64_t q_stride;
    int n_heads, rows, stages;
    float scale2;  // positive
    PrefixCut cut;
    float *slot_acc, *slot_ml;  // [2 * blocks][2][128][hs], [..][2]
    float *pre_acc, *pre_ml;    // [2 / TILES][rows of the batch * n_heads][hs], [..][2]
};

template <typename T, typename TIO, int TILES>
struct PrefixTraits {
    static constexpr bool WIDE = sizeof(TIO) == 4, F16 = std::is_same<T, __half>::value;
    static constexpr int QT = !WIDE ? 1 : F16 ? 2 : 3, PT = WIDE ? QT : 2;  // terms of Q and of P
    static constexpr float UP = !F16 ? 0.f : WIDE ? 14.f : 9.f, GROWTH = !F16 ? 8.f : WIDE ? 1.f : 6.f;  // weights up to 2^(UP + GROWTH) (weight_reference)
    static constexpr int KEYS = WIDE ? 64 : 128, STEPS = KEYS / 64, BUFFERS = STEPS;  // steps of 64 keys of a tile, buffers of a stream's scores
    static constexpr int SUB_Q = PX_ROWS * 128, SUB_K = KEYS * 128;  // bytes of 64 values of a tile's rows
    // bytes of Q's place: its terms, or 4 KB for each of the eight warps that take the sums out
    __host__ __device__ static constexpr int queries(int nd) { return QT * TILES * nd * SUB_Q > 8 * 4096 ? QT * TILES * nd * SUB_Q : 8 * 4096; }
    // instruction descriptors: f32 sums, A and B of T; B's rows along K for P V
    __host__ __device__ static constexpr uint32_t idesc(int n, int b_mn) {
        return (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(PX_ROWS >> 4) << 24);
    }
};
// 64 consecutive columns of this thread's tensor-memory lane
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&v)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
        "}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
          "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
          "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]), "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]),
          "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]), "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
          "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]), "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]),
          "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
        : "r"(taddr)
        : "memory");
}

// The first term of two weights, and what it leaves of them.  bf16's is cut off, not rounded: what is left is below 2^-7 of a weight, and the next term's rounding
// half a step of that, 2^-15 of the weight.  (Attention of 128 rows of 64 heads behind 16 000 positions, with a second term: 134 us; with the first one rounded,
// which is an instruction more per value, 153; with one term, whose rounding the results would show, 116.)
template <typename T>
__device__ __forceinline__ uint32_t first_term(float& a, float& b) {
    if constexpr (std::is_same<T, __half>::value) {
        return split_pair<T>(a, b);
    } else {
        const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
        a -= __uint_as_float(x & 0xffff0000u);
        b -= __uint_as_float(y & 0xffff0000u);
        return __byte_perm(x, y, 0x7632);
    }
}

// The softmax threads' part in bringing 128 * TILES rows of Q to shared memory, in operand layout, as terms of T.  Rows of T come by asynchronous copies,
// all of them under way at once.
template <typename T, typename TIO, int TILES>
__device__ __forceinline__ void load_queries(const PrefixParams& p, uint8_t* sq, int* s_exp, int kv, int row0, int nd) {
    using TR = PrefixTraits<T, TIO, TILES>;
    const int hs = p.pool.hs, shift = nd == 1 ? 3 : 4, tid = threadIdx.x;  // 8 or 16 threads to a row, a chunk of 8 values each
    const int ch = tid & ((1 << shift) - 1), step = 256 >> shift;
    int r = tid >> shift, t = (row0 + r) / p.group, g = (row0 + r) - t * p.group;  // row of the block, token and head of it
    const int t_step = step / p.group, g_step = step - t_step * p.group;
    const TIO* const base = (const TIO*)p.q + (int64_t)kv * p.group * hs + ch * 8;
#pragma unroll 4
    for (; r < TILES * PX_ROWS; r += step) {
        const bool real = row0 + r < p.rows && ch * 8 < hs;
        const TIO* const src = base + (int64_t)(real ? t : 0) * p.q_stride + (real ? g : 0) * hs;
        uint8_t* const dst = sq + ((r / PX_ROWS) * nd + (ch >> 3)) * TR::SUB_Q + sw128_chunk(r % PX_ROWS, ch & 7);
        if constexpr (!TR::WIDE) {
            cp_async16(dst, real ? src : (const TIO*)p.q, real);
        } else {
            float x[8] = {};
            if (real) get(src, x);
            if (TR::F16) {  // f16 terms: the row's largest value between 2^14 and 2^15, so that the steps of 2^-24 at which they stop are 2^-38 of it
                float mx = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
                for (int o = 1 << shift >> 1; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                int ex = 0;
                if (mx > 0.f && mx < INFINITY) ex = max(-100, ilogbf(mx) + 1) - 15;
                if (ch == 0) s_exp[r] = ex;
                const float f = ldexpf(1.f, -ex);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= f;
            }
#pragma unroll
            for (int k = 0; k < TR::QT; ++k) {
                uint4 w;
                w.x = split_pair<T>(x[0], x[1]);
                w.y = split_pair<T>(x[2], x[3]);
                w.z = split_pair<T>(x[4], x[5]);
                w.w = split_pair<T>(x[6], x[7]);
                *reinterpret_cast<uint4*>(dst + k * TILES * nd * TR::SUB_Q) = w;
            }
        }
        t += t_step;
        g += g_step;
        if (g >= p.group) {
            g -= p.group;
            ++t;
        }
    }
    if (!TR::WIDE) {
        cp_async_commit();
        cp_async_wait<0>();
    }
}

template <typename T, typename TIO, int TILES>
__global__ void __launch_bounds__(PX_THREADS, 1) paged_prefix_kernel(const __grid_constant__ PrefixParams p, const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_end) {
    using TR = PrefixTraits<T, TIO, TILES>;
    constexpr int KEYS = TR::KEYS;
    extern __shared__ __align__(1024) uint8_t px_raw[];
    __shared__ __align__(8) uint64_t s_kfull[PX_MAX_STAGES], s_kfree[PX_MAX_STAGES], s_vfull[PX_MAX_STAGES], s_vfree[PX_MAX_STAGES], s_mask[PX_RING], s_q, s_seg, s_s[2][2], s_p[2][2], s_o[2];  // s_s, s_p: of each buffer (a stream's softmax may be two steps ahead of its P V)
    __shared__ uint32_t s_tmem, s_valid[PX_RING][4];
    __shared__ int s_exp[TILES * PX_ROWS];
    uint8_t* const smem = px_raw + ((1024u - (smem_u32(px_raw) & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hs = p.pool.hs, nd = (hs + 63) / 64, vn = (hs + 15) / 16 * 16;
    uint8_t* const sq = smem;
    uint8_t* const sk = smem + TR::queries(nd);
    uint8_t* const sv = sk + p.stages * nd * TR::SUB_K;
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(s_kfull + i, 1);
            mbar_init(s_kfree + i, TILES);  // (the streams that read it)
            mbar_init(s_vfull + i, 1);
            mbar_init(s_vfree + i, TILES);
        }
        for (int i = 0; i < PX_RING; ++i) mbar_init(s_mask + i, 1);
        mbar_init(&s_q, 8);
        mbar_init(&s_seg, 2);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_s[i][0], 1);
            mbar_init(&s_s[i][1], 1);
            mbar_init(s_o + i, 1);
            mbar_init(&s_p[i][0], 4);
            mbar_init(&s_p[i][1], 4);
        }
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 8) tmem_alloc(&s_tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    pdl_wait();
    pdl_launch_dependents();  // (behind the wait: what follows reads the lengths before it waits itself)

    const int64_t begin = (int64_t)blockIdx.x * p.cut.share, end = min(begin + p.cut.share, p.cut.units);
    if (warp == 9) {
        // ---- copies
        bool ok = true;
        const int shift = min(p.pool.page_shift, KEYS == 128 ? 7 : 6), chunks = KEYS >> shift;  // a chunk: the map's box
        const int outside = p.pool.n_pages * p.pool.n_kv, last_page = (p.seqs.prefix_len - 1) >> p.pool.page_shift;
        // Keys run a tile ahead of the values: the products of a tile's scores come before those of the tile before with its values, and with two stages a
        // tile of values that waits for its place must not hold up the keys behind it.
        const int n = (int)(end - begin);
        int z_before = 0, y_before = 0;
        bool end_before = false;
        for (int g = 0; g <= n && ok; ++g) {
            const int stage = g % p.stages, use = g / p.stages;
            int z = outside, y = 0;
            bool at_end = false;
            if (g < n) {
                const int64_t u = begin + g;
                const int item = (int)(u / p.cut.tiles), tile = (int)(u - (int64_t)item * p.cut.tiles), kv = item / p.cut.row_tiles;
                // which keys are there: four to a lane (of one page)
                const int key = tile * KEYS + lane * 4;
                uint32_t nibble = 0;
                if (lane * 4 < KEYS && key < p.seqs.prefix_len) {
                    const int page = p.seqs.prefix_pages[key >> p.pool.page_shift];
                    if (page >= 0 && page < p.pool.n_pages) nibble = p.seqs.prefix_len - key >= 4 ? 15u : (1u << (p.seqs.prefix_len - key)) - 1u;
                }
                uint32_t word = nibble << (4 * (lane & 7));
                for (int o = 1; o < 8; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
                // a chunk of rows of one page to a lane
                const int first = tile * KEYS + (lane << shift), index = first >> p.pool.page_shift;
                int page = -1;
                if (lane < chunks && first < p.seqs.prefix_len) page = p.seqs.prefix_pages[index];
                if (page >= 0 && page < p.pool.n_pages) z = page * p.pool.n_kv + kv;
                y = first & ((1 << p.pool.page_shift) - 1);
                at_end = index == last_page;
                if (use > 0 && !mbar_wait_warp(s_kfree + stage, (uint32_t)((use - 1) & 1))) {
                    ok = false;
                    break;
                }
                if ((lane & 7) == 0) s_valid[g % PX_RING][lane >> 3] = word;
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(s_mask + g % PX_RING);
                    mbar_arrive_expect_tx(s_kfull + stage, (uint32_t)(nd * TR::SUB_K));
                }
                __syncwarp();
                if (lane < chunks)
                    for (int d = 0; d < nd; ++d) tma_load_3d(sk + (stage * nd + d) * TR::SUB_K + (lane << shift) * 128, &map_k, 64 * d, y, z, s_kfull + stage);
            }
            if (g > 0) {
                const int vs = (g - 1) % p.stages, vu = (g - 1) / p.stages;
                if (vu > 0 && !mbar_wait_warp(s_vfree + vs, (uint32_t)((vu - 1) & 1))) {
                    ok = false;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(s_vfull + vs, (uint32_t)(nd * TR::SUB_K));
                __syncwarp();
                if (lane < chunks)
                    for (int d = 0; d < nd; ++d)
                        tma_load_3d(sv + (vs * nd + d) * TR::SUB_K + (lane << shift) * 128, end_before ? &map_end : &map_v, 64 * d, y_before, z_before, s_vfull + vs);
            }
            z_before = z;
            y_before = y;
            end_before = at_end;
        }
        if (!ok)
            for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies in flight land within microseconds
    } else if (warp >= 8) {
        // ---- products of a stream
        // The warp goes through its loop together and one thread of it issues: descriptors are uniform, stages and phases are counted, not divided for.  (By a thread
        // that had the loop for itself a product took 110 cycles to issue, twice its length.)
        const int i = warp == 8 ? 0 : 1;
        const bool leader = elect_one();
        const uint32_t idesc_s = TR::idesc(64, 0), idesc_o = TR::idesc(vn, 1), stage_step = (uint32_t)(nd * TR::SUB_K) >> 4;
        const uint64_t desc_q = umma_desc_sw128(sq + (TILES == 2 ? i : 0) * nd * TR::SUB_Q, 0), desc_k = umma_desc_sw128(sk, 0), desc_v = umma_desc_sw128_mn(sv, 0, TR::SUB_K);
        const uint32_t ds = tmem + (uint32_t)(i * 128), dout = tmem + 256 + (uint32_t)(i * 128);
        bool ok = true;
        int g = 0, segment = 0;
        struct Place {  // in a ring
            int stage;
            uint32_t phase;
        } k = {0, 0}, v = {0, 0};
        uint32_t before = 0;  // steps of the segments before
        auto advance = [&](Place& at) {
#pragma unroll
            for (int j = 0; j < (TILES == 2 ? 1 : 2); ++j)
                if (++at.stage == p.stages) {
                    at.stage = 0;
                    at.phase ^= 1u;
                }
        };
        auto qk = [&](uint32_t n) {  // scores of step n
            const uint32_t buffer = (before + n) % TR::BUFFERS, half = n % TR::STEPS;
            if (half == 0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(s_kfull + k.stage, k.phase));
            if (!ok) return;
            tc_fence_after();
            const uint64_t kd = desc_k + (uint32_t)k.stage * stage_step + half * (64 * 128 >> 4);
            const uint32_t d = ds + buffer * 64;
#pragma unroll
            for (int t = TR::QT - 1; t >= 0; --t) {  // (small terms first)
                const uint64_t qd = desc_q + (uint32_t)(t * TILES * nd) * (uint32_t)(TR::SUB_Q >> 4);
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
                    if (sub < nd && leader) {  // (values behind a head's end are zeros)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            umma_f16(d, qd + (uint32_t)(sub * (TR::SUB_Q >> 4) + kk * 2), kd + (uint32_t)(sub * (TR::SUB_K >> 4) + kk * 2), idesc_s, t == TR::QT - 1 && sub == 0 && kk == 0 ? 0u : 1u);
                    }
            }
            if (leader) umma_commit(&s_s[i][buffer]);
            if (half == TR::STEPS - 1) {
                if (leader) umma_commit(s_kfree + k.stage);
                advance(k);
            }
        };
        auto pv = [&](uint32_t n) {
            const uint32_t c = before + n, buffer = c % TR::BUFFERS, half = n % TR::STEPS;
            const uint64_t vd = desc_v + (uint32_t)v.stage * stage_step + half * (64 * 128 >> 4);
            const uint32_t a = ds + buffer * 64;
            if (half == 0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(s_vfull + v.stage, v.phase));
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_p[i][buffer], c / TR::BUFFERS & 1u));
            if (!ok) return;
            tc_fence_after();
            if (leader) {
#pragma unroll
                for (int t = TR::PT - 1; t >= 0; --t)
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        umma_f16_at(dout, a + (uint32_t)(t * 32 + kk * 8), vd + (uint32_t)(kk * (2048 >> 4)), idesc_o, t < TR::PT - 1 || kk > 0 ? 1u : n > 0 ? 1u : 0u);
                umma_commit(s_o + i);
            }
            if (half == TR::STEPS - 1) {
                if (leader) umma_commit(s_vfree + v.stage);
                advance(v);
            }
        };
        for (int64_t u = begin; u < end && ok; ++segment) {
            const int item = (int)(u / p.cut.tiles), tiles = (int)min((int64_t)p.cut.tiles - (u - (int64_t)item * p.cut.tiles), end - u);
            const uint32_t n = (uint32_t)(TR::STEPS * (TILES == 2 ? tiles : (tiles + 1 - i) / 2));  // steps of this stream
            const int first = TILES == 2 ? g : g + i;
            k = v = {first % p.stages, (uint32_t)(first / p.stages & 1)};
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_q, (uint32_t)(segment & 1)));
#pragma unroll 1
            for (uint32_t t = 0; t < n + TR::BUFFERS && ok; ++t) {  // P V of a step, then Q K^T of the one that gets its buffer
                if (t >= TR::BUFFERS) pv(t - TR::BUFFERS);
                if (ok && t < n) qk(t);
            }
            before += n;
            if (ok && leader) umma_commit(&s_seg);
            g += tiles;
            u += tiles;
        }
    } else {
        // ---- softmax: a thread per row of its stream
        const int i = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + lanes + (uint32_t)(i * 128), to = tmem + 256 + lanes + (uint32_t)(i * 128);
        bool ok = true;
        int g = 0, segment = 0, ns = 0;
        for (int64_t u = begin; u < end; ++segment) {
            const int item = (int)(u / p.cut.tiles), first_tile = (int)(u - (int64_t)item * p.cut.tiles), n = (int)min((int64_t)p.cut.tiles - first_tile, end - u);
            const int kv = item / p.cut.row_tiles, row_tile = item - kv * p.cut.row_tiles;
            load_queries<T, TIO, TILES>(p, sq, s_exp, kv, row_tile * TILES * PX_ROWS, nd);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_q);
            float sc = p.scale2;
            if (TR::WIDE && TR::F16) {
                asm volatile("bar.sync 1, 256;" ::: "memory");  // (the row's exponent is another thread's)
                sc = ldexpf(sc, s_exp[TILES == 2 ? i * PX_ROWS + r : r]);
            }
            float m = -INFINITY, l = 0.f;
            bool some = false;
            for (int t = TILES == 2 ? 0 : i; t < n; t += TILES == 2 ? 1 : 2) {
                const int gt = g + t;
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(s_mask + gt % PX_RING, (uint32_t)(gt / PX_RING & 1)));
#pragma unroll 1
                for (int step = 0; step < TR::STEPS; ++step, ++ns) {
                    const int buffer = ns % TR::BUFFERS;
                    const uint32_t tb = ts + (uint32_t)(buffer * 64);
                    if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_s[i][buffer], (uint32_t)(ns / TR::BUFFERS & 1)));
                    tc_fence_after();
                    float x[64];
                    tmem_load(tb, x);
                    const uint32_t v0 = s_valid[gt % PX_RING][2 * step], v1 = s_valid[gt % PX_RING][2 * step + 1];
                    if ((v0 & v1) != ~0u) {
#pragma unroll
                        for (int k = 0; k < 64; ++k) x[k] = (k < 32 ? v0 : v1) >> (k & 31) & 1 ? x[k] : -INFINITY;
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 64; k += 2) m4[k >> 1 & 3] = fmaxf(fmaxf(x[k], x[k + 1]), m4[k >> 1 & 3]);
                    float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sc;
                    if (TR::UP != 0.f) mx = weight_reference(mx, TR::UP);
                    if (!some) {
                        m = mx;
                    } else if (__any_sync(0xffffffffu, mx > m + TR::GROWTH)) {
                        const float mn = fmaxf(mx, m), corr = m == -INFINITY ? 0.f : exp2_approx(m - mn);  // (a row that has seen nothing has sums of zero)
                        l *= corr;
                        m = mn;
                        if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(s_o + i, (uint32_t)((ns - 1) & 1)));  // the sums of the step before are there
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < vn; c += 16) {
                            float o[16];
                            tmem_ld16f(to + (uint32_t)c, o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] *= corr;
                            tmem_st16f(to + (uint32_t)c, o);
                        }
                    }
                    some = true;
                    const float use = m == -INFINITY ? 0.f : m;
                    float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 64; c += 16) {  // (the exponentials of some while others become terms)
#pragma unroll
                        for (int k = c; k < c + 16; ++k) {
                            x[k] = exp2_approx(fmaf(x[k], sc, -use));
                            l4[k & 3] += x[k];
                        }
#pragma unroll
                        for (int t2 = 0; t2 < TR::PT; ++t2) {
                            uint32_t w[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) w[k] = t2 == 0 ? first_term<T>(x[c + 2 * k], x[c + 2 * k + 1]) : split_pair<T>(x[c + 2 * k], x[c + 2 * k + 1]);
                            tmem_st8(tb + (uint32_t)(t2 * 32 + c / 2), w);  // (in the place of the scores, which have been read)
                        }
                    }
                    l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_p[i][buffer]);
                }
            }
            // the segment's products are all done: this row's sums to the workspace
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_seg, (uint32_t)(segment & 1)));
            tc_fence_after();
            if (l != l && m == -INFINITY) m = 0.f;  // scores that are no numbers are not an empty row
            if (!ok) {
                m = 0.f;
                l = NAN;
            }
            const int row = row_tile * TILES * PX_ROWS + (TILES == 2 ? i * PX_ROWS : 0) + r;
            const bool whole = n == p.cut.tiles, real = row < p.rows;
            int64_t at;
            if (whole) {
                const int t = row / p.group;
                at = (TILES == 1 ? (int64_t)i * p.cut.whole_rows : 0) + (int64_t)t * p.n_heads + kv * p.group + row - t * p.group;
            } else {
                at = ((int64_t)(2 * blockIdx.x + (first_tile == 0 ? 1 : 0)) * 2 + i) * PX_ROWS + r;
            }
            if (real) *reinterpret_cast<float2*>((whole ? p.pre_ml : p.slot_ml) + at * 2) = make_float2(m, l);
            // The sums go through shared memory, in Q's place, so that a row's 32 values are written together: 4 KB per warp, 16-byte chunks swizzled.
            if (some) {  // (the same for the whole warp)
                float* const acc = whole ? p.pre_acc : p.slot_acc;
                uint8_t* const st = sq + warp * 4096;
#pragma unroll 1
                for (int c = 0; c < hs; c += 32) {
                    float o[32];
                    tmem_ld32f(to + (uint32_t)c, o);
#pragma unroll
                    for (int e = 0; e < 8; ++e) *reinterpret_cast<float4*>(st + sw128_chunk(lane, e)) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int rr = e * 4 + (lane >> 3), ch = lane & 7;
                        const int64_t to_row = __shfl_sync(0xffffffffu, real ? at : -1, rr);
                        if (to_row >= 0 && c + ch * 4 < hs) *reinterpret_cast<float4*>(acc + to_row * hs + c + ch * 4) = *reinterpret_cast<const float4*>(st + sw128_chunk(rr, ch));
                    }
                    __syncwarp();
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");  // (the next segment's Q comes where other warps' sums may be still)
            tc_fence_before();  // (the next segment's products overwrite the sums)
            g += n;
            u += n;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) tmem_dealloc(tmem, 512);
}

}  // namespace l2b
