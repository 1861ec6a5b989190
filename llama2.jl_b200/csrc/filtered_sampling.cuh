// The next token of each row of logits by temperature, top-k, top-p and min-p from a given random number.
//   w_i = exp((x_i - max) / T);  order: larger x first, of equal ones the lower index first.
//   top-k keeps the first k;  top-p keeps those before which less than p of the mass of what top-k keeps lies;  min-p keeps w_i >= min_p;  the first
//   is always kept.  The token is the first, by index, at which the kept tokens' cumulated mass exceeds u times their whole.
//
// A cluster of up to eight blocks holds a row in its shared memory, read once; every pass after that is over shared memory.  Masses are whole numbers of
// 2^-44 of the largest weight (weights computed in 64 bits), so that sums do not depend on their order and no cut or choice hangs on the blocks or on atomics.
//   top-k up to FS_FAST: every block takes its share of the k-th place among its threads' maxima, so that the lowest of the blocks' values has at least k
//     values above it; the few that are no smaller are brought together, and everything else happens among those.
//   other cuts: equal bins of the distance from the maximum are counted, or weighed; only the bin with the k-th value, or the nucleus' border, is listed and
//     ordered, by counting.  More than FS_LIST values in one bin (many equal logits): bisection on (value, index), a pass per bit.
//   the choice: masses of stretches of the row, then inside the stretch that holds it.
// What every block needs it works out for itself from the others' shared memory: a barrier of the cluster costs more than that.
// A pass that weighs all logits is bound by 64-bit arithmetic, one over a few candidates by the barriers; the logits' read is the floor.
#pragma once
#include <cooperative_groups.h>

#include "paged_append.cuh"

namespace l2b {

constexpr int FS_THREADS = 512, FS_WARPS = FS_THREADS / 32, FS_BINS = 1024, FS_LIST = 1024, FS_FAST = 512, FS_CLUSTER = 8, FS_TABLE = 128;
constexpr int FS_SLICE = 48 * 1024;  // most logits of a block
constexpr double FS_ONE = 17592186044416.0;  // 2^44

struct SampleParams {
    const void* logits;
    int64_t stride;
    int vocab, slice, cluster;
    const float *temperature, *top_p, *min_p;  // null: 1, no cut, no cut
    const int* top_k;                          // null: no cut
    const double* uniform;
    int* tokens;
    float* probs;  // may be null
};

struct SampleShared {
    union {
        struct {
            uint32_t low[FS_BINS], high[FS_BINS];  // of each bin: the count in `low`, or the mass
        };
        uint64_t w[FS_LIST];  // weights of `all`, once all blocks have read the bins (a gathering's barrier is behind that)
    };
    uint64_t list[FS_LIST];
    uint64_t all[FS_LIST];                 // the lists of all blocks
    double table[FS_TABLE];                // 2^(-i / FS_TABLE)
    uint64_t sums[FS_WARPS];
    float wmax[FS_WARPS], wmin[FS_WARPS], tmax[FS_THREADS];
    uint32_t widx[FS_WARPS], wcnt[FS_WARPS];
    // what other blocks read
    float max, min, tau;
    uint32_t idx, usable, listed;
    uint64_t total[2];
    // found by one thread, used by all
    int bin;
    uint32_t survivors, choice;
    uint64_t before, found;
};

__device__ __forceinline__ uint32_t ordered_bits(float x) {  // larger value, larger number; -0 and 0 are equal
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) { return (uint64_t)ordered_bits(x) << 32 | (0xffffffffu - index); }

struct SampleRow {
    float top;
    double shift, rate, floor_t;  // w = 2^-t, t = shift - x * rate; floor_t: no weight beyond
    double min_p;
    uint64_t first;  // key of the first token: always kept
    const double* table;
    // 2^-t: t to the nearest 1/128 from the table, the rest (a = rest * ln 2 up to 0.0027) by the exponential series up to a^4 / 24; a^5 / 120 is 1.2e-15.
    __device__ __forceinline__ double weight(float x) const {
        if (x == top) return 1.0;
        const double t = fma(-(double)x, rate, shift);
        if (!(t < floor_t)) return 0.0;  // (also: infinite minus infinite)
        constexpr double magic = 6755399441055744.0 / FS_TABLE;  // 1.5 * 2^52 / 128: the sum's last bit is 1/128
        const double u = t + magic;
        const int k = max(0, (int)(__double_as_longlong(u) & 0xffffffff));
        const double a = (t - (u - magic)) * -0.6931471805599453;
        const double q = fma(a, fma(a, fma(a, fma(a, 1.0 / 24, 1.0 / 6), 0.5), 1.0), 1.0) * table[k & (FS_TABLE - 1)];
        return __longlong_as_double(__double_as_longlong(q) - ((long long)(k / FS_TABLE) << 52));  // (2^-46 at least)
    }
    // In units of 2^-44, to the nearest: the last bits of w + 2^8.
    static __device__ __forceinline__ uint64_t units(double w) { return (uint64_t)(__double_as_longlong(w + 256.0) - __double_as_longlong(256.0)); }
    __device__ __forceinline__ uint64_t mass(float x) const { return units(weight(x)); }
    // of a value that the order keeps
    __device__ __forceinline__ uint64_t kept_mass(float x, uint64_t key) const {
        const double w = weight(x);
        return w >= min_p || key == first ? units(w) : 0;
    }
};

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum over the block, for all threads.
__device__ __forceinline__ uint64_t block_total(uint64_t v, SampleShared& s) {
    v = warp_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.sums[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < FS_WARPS; ++w) v += s.sums[w];
    return v;
}
// Sum of the threads before this one.
__device__ __forceinline__ uint64_t block_before(uint64_t v, SampleShared& s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t inc = v;
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) s.sums[warp] = inc;
    __syncthreads();
    uint64_t b = inc - v;
    for (int w = 0; w < warp; ++w) b += s.sums[w];
    return b;
}

// Exact mass of a bin: two 32-bit words, the carry by hand.
__device__ __forceinline__ void add_mass(SampleShared& s, int bin, uint64_t w) {
    const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.low[bin], lo), hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
    if (hi) atomicAdd(&s.high[bin], hi);
}

// For every one of n keys in s.all: how many are above it, and their mass.  Several threads share a key when there are few: `lanes` of them, and all get the
// sums.  body(e, i, place, above): i = the key's number, n or more for none; e counts this thread's keys.
template <class Body>
__device__ __forceinline__ void for_each_above(SampleShared& s, int n, Body&& body) {
    int lanes = 16;
    while (lanes > 1 && FS_THREADS / lanes < n) lanes /= 2;
    const int q = threadIdx.x % lanes;
#pragma unroll
    for (int e = 0; e < FS_LIST / FS_THREADS; ++e) {
        const int i = (int)threadIdx.x / lanes + e * (FS_THREADS / lanes);
        if (e > 0 && FS_THREADS / lanes >= n) break;  // (the same for all threads)
        const uint64_t key = i < n ? s.all[i] : ~0ull;
        uint32_t place = 0;
        uint64_t above = 0;
#pragma unroll 4
        for (int j = q; j < n; j += lanes) {
            const bool yes = s.all[j] > key;
            place += yes;
            above += yes ? s.w[j] : 0;
        }
        for (int o = 1; o < lanes; o <<= 1) {
            place += __shfl_xor_sync(0xffffffffu, place, o);
            above += __shfl_xor_sync(0xffffffffu, above, o);
        }
        body(e, i, key, place, above, q == 0);
    }
}

template <typename T>
__global__ void __launch_bounds__(FS_THREADS) filtered_sample_kernel(const __grid_constant__ SampleParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) float fs_x[];
    __shared__ SampleShared s;
    const cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)blockIdx.x % p.cluster, row = (int)(blockIdx.x / p.cluster);
    const int first = rank * p.slice, n = max(0, min(p.slice, p.vocab - first));
    if (tid < FS_TABLE) s.table[tid] = exp2(-(double)tid / FS_TABLE);
    for (int i = tid; i < FS_BINS; i += FS_THREADS) s.low[i] = s.high[i] = 0;
    if (tid == 0) s.survivors = 0;
    pdl_wait();
    const float temperature = p.temperature ? p.temperature[row] : 1.f;
    const int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p && p.min_p[row] > 0.f ? p.min_p[row] : 0.f;
    double u = p.uniform[row];

    // the slice, its maximum (first of equals), its smallest finite value and how many values are choices at all
    float mx = -INFINITY, mn = INFINITY;
    uint32_t mi = 0xffffffffu, usable = 0;
    auto take = [&](int i, float x) {
        x = x > -INFINITY ? x + 0.f : -INFINITY;  // no number: no choice
        fs_x[i] = x;
        if (x > mx) {
            mx = x;
            mi = (uint32_t)(first + i);
        }
        if (x > -INFINITY) {
            ++usable;
            mn = fminf(mn, x);
        }
    };
    const T* const src = (const T*)p.logits + row * p.stride + first;
    constexpr int V = 16 / sizeof(T);
    const int nv = ((uintptr_t)src & 15) == 0 ? n / V : 0;
#pragma unroll 4
    for (int i = tid; i < nv; i += FS_THREADS) {
        float x[V];
        get(src + i * V, x);
#pragma unroll
        for (int e = 0; e < V; ++e) take(i * V + e, x[e]);
    }
#pragma unroll 4
    for (int i = nv * V + tid; i < n; i += FS_THREADS) take(i, to_f32(src[i]));
    const float own_max = mx;
    for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, mx, o);
        const uint32_t i = __shfl_xor_sync(0xffffffffu, mi, o);
        if (v > mx || (v == mx && i < mi)) {
            mx = v;
            mi = i;
        }
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        usable += __shfl_xor_sync(0xffffffffu, usable, o);
    }
    if (lane == 0) {
        s.wmax[warp] = mx;
        s.widx[warp] = mi;
        s.wmin[warp] = mn;
        s.wcnt[warp] = usable;
    }
    __syncthreads();
    float weakest = INFINITY;
    for (int w = 0; w < FS_WARPS; ++w) weakest = fminf(weakest, s.wmax[w]);
    if (tid == 0) {
        mx = -INFINITY;
        mn = INFINITY;
        mi = 0xffffffffu;
        usable = 0;
        for (int w = 0; w < FS_WARPS; ++w) {
            if (s.wmax[w] > mx || (s.wmax[w] == mx && s.widx[w] < mi)) {
                mx = s.wmax[w];
                mi = s.widx[w];
            }
            mn = fminf(mn, s.wmin[w]);
            usable += s.wcnt[w];
        }
        s.max = mx;
        s.idx = mi;
        s.min = mn;
        s.usable = usable;
        s.listed = 0;
        s.tau = -INFINITY;
    }
    // The block's share of the k-th place: the value at that place among its threads' maxima (of up to 16: only those as large as the weakest warp's
    // count, there are 16 of them at least).
    const bool fast = k > 1 && k <= FS_FAST;
    if (fast) {
        const int place = (k + p.cluster - 1) / p.cluster - 1;
        const bool in = place >= FS_WARPS || own_max >= weakest;
        const unsigned v = __ballot_sync(0xffffffffu, in);
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&s.survivors, __popc(v));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(v & ((1u << lane) - 1u));
        if (in) s.tmax[at] = own_max;
        __syncthreads();
        const int m = (int)s.survivors;
        if (tid < m) {
            const float mine = s.tmax[tid];
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < m; ++j) above += s.tmax[j] > mine || (s.tmax[j] == mine && j < tid);
            if (above == place) s.tau = mine;
        }
    }
    cluster.sync();
    float tau = INFINITY;
    mx = -INFINITY;
    mn = INFINITY;
    mi = 0xffffffffu;
    usable = 0;
    for (int b = 0; b < p.cluster; ++b) {
        const SampleShared* o = cluster.map_shared_rank(&s, b);
        const float v = o->max;
        if (v > mx) {  // (the lower index first: blocks hold ascending ranges)
            mx = v;
            mi = o->idx;
        }
        mn = fminf(mn, o->min);
        tau = fminf(tau, o->tau);
        usable += o->usable;
    }

    const bool has_k = k > 0 && (uint32_t)k < usable, has_p = top_p < 1.f;
    if (usable == 0 || !(temperature > 0.f) || k == 1 || top_p <= 0.f) {  // nothing to choose from, or to choose
        if (rank == 0 && tid == 0) {
            p.tokens[row] = usable ? (int)mi : -1;
            if (p.probs) p.probs[row] = usable ? 1.f : 0.f;
        }
        cluster.sync();  // (nobody leaves while its shared memory is read)
        return;
    }
    SampleRow r;
    r.top = mx;
    r.rate = 1.4426950408889634 / (double)temperature;
    r.shift = (double)mx * r.rate;
    r.floor_t = 46.0;
    r.min_p = (double)min_p;
    r.first = order_key(mx, mi);
    r.table = s.table;
    u = u > 0.0 ? fmin(u, 1.0) : 0.0;
    // the last of the mass counts as not reached: u * whole rounds to at most whole, and the token is there where the sum exceeds it
    auto border = [&](uint64_t whole) { return min((uint64_t)(u * (double)whole), whole - 1); };
    const float span = fminf(mx - mn, 32.f * temperature);
    const float per = span > 1e-30f ? (float)FS_BINS / span : 1e30f;  // (an infinite span: everything in bin 0)
    auto bin_of = [&](float x) { return min(FS_BINS - 1, (int)((mx - x) * per)); };
    uint64_t cut = 0;  // key of the last that is kept

    // Values of one kind, listed by every block and brought together.  Returns how many there are (more than FS_LIST: no list).  everyone: for all
    // blocks, else for block 0.
    auto gather = [&](bool everyone, auto&& wanted) -> uint32_t {
        if (tid == 0) s.listed = 0;
        __syncthreads();
        for (int i0 = 0; i0 < n; i0 += FS_THREADS) {
            const int i = i0 + tid;
            const bool yes = i < n && fs_x[i] > -INFINITY && wanted(fs_x[i], (uint32_t)(first + i));
            const unsigned v = __ballot_sync(0xffffffffu, yes);
            if (v) {
                uint32_t at = 0;
                if (lane == 0) at = atomicAdd(&s.listed, __popc(v));
                at = __shfl_sync(0xffffffffu, at, 0) + __popc(v & ((1u << lane) - 1u));
                if (yes && at < FS_LIST) s.list[at] = order_key(fs_x[i], (uint32_t)(first + i));
            }
        }
        cluster.sync();
        uint32_t all = 0, of[FS_CLUSTER];
#pragma unroll
        for (int b = 0; b < FS_CLUSTER; ++b) {
            of[b] = b < p.cluster ? cluster.map_shared_rank(&s, b)->listed : 0;
            all += of[b];
        }
        if (all <= FS_LIST && (everyone || rank == 0)) {
            for (uint32_t i = tid; i < all; i += FS_THREADS) {
                uint32_t b = 0, at = i;
#pragma unroll
                for (int c = 0; c < FS_CLUSTER - 1; ++c)
                    if (b == (uint32_t)c && at >= of[c]) {
                        at -= of[c];
                        ++b;
                    }
                const uint64_t key = cluster.map_shared_rank(&s, b)->list[at];
                s.all[i] = key;
                s.w[i] = r.mass(from_ordered((uint32_t)(key >> 32)));
            }
            __syncthreads();
        }
        return all;
    };
    // The smallest key c with measure(keys above c) below `most`: what is kept is c and all above it.  A pass over the row per bit.
    auto bisect = [&](auto&& measure, double most) -> uint64_t {
        uint64_t lo = (uint64_t)ordered_bits(mn) << 32, hi = r.first;  // holds at hi: nothing is above it
        int turn = 0;
        while (lo < hi) {
            const uint64_t mid = lo + (hi - lo) / 2;
            uint64_t v = 0;
            for (int i = tid; i < n; i += FS_THREADS) {
                const uint64_t key = order_key(fs_x[i], (uint32_t)(first + i));
                if (fs_x[i] > -INFINITY && key > mid) v += measure(fs_x[i], key);
            }
            v = block_total(v, s);
            if (tid == 0) s.total[turn] = v;
            cluster.sync();
            uint64_t all = 0;
            for (int b = 0; b < p.cluster; ++b) all += cluster.map_shared_rank(&s, b)->total[turn];
            turn ^= 1;  // (the other slot: a block may be a step ahead)
            if ((double)all < most) hi = mid;
            else lo = mid + 1;
        }
        cluster.sync();
        return lo;
    };
    // The bin at which the running measure (counts, or masses) reaches `most`, and the measure before it and with it; the last bin, which is not measured, has the rest.
    auto reach = [&](double most) {
        uint64_t c[FS_BINS / FS_THREADS], sum = 0;
#pragma unroll
        for (int e = 0; e < FS_BINS / FS_THREADS; ++e) {
            c[e] = 0;
            const int bin = tid * (FS_BINS / FS_THREADS) + e;
            for (int b = 0; b < p.cluster; ++b) {
                const SampleShared* o = cluster.map_shared_rank(&s, b);
                c[e] += (uint64_t)o->high[bin] << 32;
                c[e] += o->low[bin];
            }
            sum += c[e];
        }
        uint64_t before = block_before(sum, s);
        if (tid == FS_THREADS - 1) {
            s.bin = FS_BINS - 1;
            s.before = before + sum;
            s.found = ~0ull;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < FS_BINS / FS_THREADS; ++e) {
            if ((double)before < most && (double)(before + c[e]) >= most) {
                s.bin = tid * (FS_BINS / FS_THREADS) + e;
                s.before = before;
                s.found = before + c[e];
            }
            before += c[e];
        }
        __syncthreads();
    };

    if (has_k) {
        uint32_t m = FS_LIST + 1;
        if (fast) m = gather(false, [&](float x, uint32_t) { return x >= tau; });
        if (m <= FS_LIST) {
            // everything that is kept is among these
            if (rank == 0) {
                constexpr int E = FS_LIST / FS_THREADS;
                uint64_t above[E] = {}, key[E] = {}, w[E] = {}, mass_k = 0;
                uint32_t place[E] = {};
                bool mine[E] = {};  // (one of the threads that share a key)
                for_each_above(s, (int)m, [&](int e, int i, uint64_t ke, uint32_t pl, uint64_t ab, bool one) {
                    mine[e] = one && i < (int)m;
                    key[e] = ke;
                    place[e] = pl;
                    above[e] = ab;
                    w[e] = mine[e] && pl < (uint32_t)k ? s.w[i] : 0;
                    mass_k += w[e];
                });
                const double most = (double)top_p * (double)block_total(mass_k, s);
                uint64_t whole = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const bool keep = mine[e] && place[e] < (uint32_t)k && (!has_p || (double)above[e] < most || key[e] == r.first);
                    w[e] = keep ? r.kept_mass(from_ordered((uint32_t)(key[e] >> 32)), key[e]) : 0;
                    whole += w[e];
                }
                whole = block_total(whole, s);  // (its barriers: everyone has read s.all and s.w)
                // the kept ones again, ordered by index: keys with the index in front
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (mine[e]) {
                        s.all[place[e]] = w[e] ? (key[e] & 0xffffffffu) : 0;  // (higher for a lower index)
                        s.w[place[e]] = w[e];
                    }
                __syncthreads();
                const uint64_t most_u = border(whole);
                for_each_above(s, (int)m, [&](int e, int i, uint64_t ke, uint32_t, uint64_t ab, bool one) {
                    if (one && i < (int)m && ke && ab <= most_u && most_u < ab + s.w[i]) {  // (of one key only)
                        p.tokens[row] = (int)(0xffffffffu - (uint32_t)ke);
                        if (p.probs) p.probs[row] = (float)((double)s.w[i] / (double)whole);
                    }
                });
            }
            cluster.sync();
            return;
        }
        for (int i = tid; i < n; i += FS_THREADS) {
            const int b = fs_x[i] > -INFINITY ? bin_of(fs_x[i]) : FS_BINS - 1;
            if (b < FS_BINS - 1) atomicAdd(&s.low[b], 1u);
        }
        cluster.sync();
        reach((double)k);
        const int bk = s.bin;
        const uint32_t ahead = (uint32_t)s.before, upto = s.found != ~0ull ? (uint32_t)s.found : usable;
        if (upto - ahead <= FS_LIST) {
            m = gather(true, [&](float x, uint32_t) { return bin_of(x) == bk; });
            for_each_above(s, (int)m, [&](int, int i, uint64_t key, uint32_t place, uint64_t, bool one) {
                if (one && i < (int)m && ahead + place == (uint32_t)k - 1) s.found = key;
            });
            __syncthreads();
            cut = s.found;
        } else {
            cut = bisect([](float, uint64_t) { return (uint64_t)1; }, (double)k);
        }
        if (has_p) {
            cluster.sync();  // (all have read the counts)
            for (int i = tid; i < FS_BINS; i += FS_THREADS) s.low[i] = s.high[i] = 0;
            __syncthreads();
        }
    }

    if (has_p) {
        uint64_t sum = 0;
        for (int i = tid; i < n; i += FS_THREADS) {
            const float x = fs_x[i];
            if (x > -INFINITY && order_key(x, (uint32_t)(first + i)) >= cut) {
                const uint64_t w = r.mass(x);
                const int b = bin_of(x);
                sum += w;
                if (w && b < FS_BINS - 1) add_mass(s, b, w);
            }
        }
        sum = block_total(sum, s);
        if (tid == 0) s.total[0] = sum;
        cluster.sync();
        uint64_t whole = 0;
        for (int b = 0; b < p.cluster; ++b) whole += cluster.map_shared_rank(&s, b)->total[0];
        const double most = (double)top_p * (double)whole;
        reach(most);
        const int bp = s.bin;
        const uint64_t ahead = s.before;
        const uint32_t m = gather(true, [&](float x, uint32_t index) { return bin_of(x) == bp && order_key(x, index) >= cut; });
        if (m <= FS_LIST) {
            if (tid == 0) s.found = r.first;  // (the first is always kept)
            __syncthreads();
            for_each_above(s, (int)m, [&](int, int i, uint64_t key, uint32_t, uint64_t above, bool one) {
                if (one && i < (int)m && (double)(ahead + above) < most) atomicMin((unsigned long long*)&s.found, (unsigned long long)key);
            });
            __syncthreads();
            cut = max(cut, s.found);
        } else {
            const uint64_t old = cut;
            cut = max(old, bisect([&](float x, uint64_t key) { return key >= old ? r.mass(x) : (uint64_t)0; }, most));
        }
    }

    // the choice among all that is kept: masses per warp's stretch of the slice, then inside the stretch that holds it
    if (min_p > 0.f) r.floor_t = fmin(r.floor_t, fmax(0.0, 1e-6 - log2((double)min_p)));  // (a little beyond min_p: the comparison is made on the weight)
    const int stretch = (p.slice + FS_WARPS - 1) / FS_WARPS;
    auto kept = [&](int i) -> uint64_t {
        const float x = fs_x[i];
        if (!(x > -INFINITY)) return 0;
        const uint64_t key = order_key(x, (uint32_t)(first + i));
        return key >= cut ? r.kept_mass(x, key) : 0;
    };
    const int lo = min(n, warp * stretch), hi = min(n, lo + stretch);
    uint64_t sum = 0;
    for (int i = lo + lane; i < hi; i += 32) sum += kept(i);
    sum = warp_sum64(sum);
    __syncthreads();
    if (lane == 0) s.sums[warp] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < FS_WARPS; ++w) sum += s.sums[w];
    if (tid == 0) s.total[1] = sum;
    cluster.sync();
    uint64_t whole = 0, ahead = 0;
    for (int b = 0; b < p.cluster; ++b) {
        const uint64_t t = cluster.map_shared_rank(&s, b)->total[1];
        whole += t;
        ahead += b < rank ? t : 0;
    }
    const uint64_t most_u = border(whole);
    if (ahead <= most_u && most_u < ahead + sum) {  // here (one block of the cluster, and all of its threads)
        int w = 0;
        while (ahead + s.sums[w] <= most_u) ahead += s.sums[w++];
        const int l = min(n, w * stretch), h = min(n, l + stretch), each = (stretch + FS_THREADS - 1) / FS_THREADS;
        const int a = min(h, l + tid * each), z = min(h, a + each);
        uint64_t mine = 0;
        for (int i = a; i < z; ++i) mine += kept(i);
        uint64_t run = ahead + block_before(mine, s);
        if (run <= most_u && most_u < run + mine) {
            for (int i = a; i < z; ++i) {
                const uint64_t m = kept(i);
                if (run + m > most_u) {
                    p.tokens[row] = first + i;
                    if (p.probs) p.probs[row] = (float)((double)m / (double)whole);
                    break;
                }
                run += m;
            }
        }
    }
    cluster.sync();
}

}  // namespace l2b
