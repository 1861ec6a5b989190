// The next token of each row of logits by temperature, top-k, top-p and min-p from a given random number.
//   w_i = exp((x_i - max) / T);  order: larger x first, of equal ones the lower index first.
//   top-k keeps the first k;  top-p keeps those before which less than p of the mass of what top-k keeps lies;  min-p keeps w_i >= min_p;  the first
//   is always kept.  The token is the first, by index, at which the kept tokens' cumulated mass exceeds u times their whole.
//
// A cluster of up to eight blocks holds a row in its shared memory, read once; every pass after that is over shared memory.  Masses are whole numbers of
// 2^-44 of the largest weight (weights computed in 64 bits), so that sums do not depend on their order and no cut or choice hangs on the blocks or on atomics.
// (The whole of a row is below 2^63 then.  Weights below half a unit are none; a border may lie off by half a unit a logit, 1.1e-8 of the largest weight for 393 216.)
//   top-k up to FS_FAST: every block takes its share of the k-th place among its threads' maxima, so that the lowest of the blocks' values has at least k
//     values that are no smaller; those few go to the first block, which does the rest alone while the others leave.
//   other cuts: equal bins of the distance from the maximum are counted, or weighed; only the bin with the k-th value, or the nucleus' border, is listed and
//     ordered, by counting.  More than FS_LIST values in one bin (many equal logits): bisection on (value, index), a pass per bit.
//   the choice: masses of stretches of the row, then inside the stretch that holds it.
// Blocks write what the others need into the others' shared memory in front of a barrier, so that it is at hand behind it; nothing is fetched from a block
// after the last barrier, so blocks leave at once.
// Passes that compare take four logits at a time.  With a cut below it the kept logits are collected 32 at a time before they are weighed.  A pass that weighs all
// logits is bound by issue slots: 200 rows of 32 000 logits with top-p alone are 181 warp instructions per 32 logits, the ALU 44 % and the 64-bit pipe 12 % busy; the 400
// blocks find 296 places, so that the schedulers issue 65 % of the time and the busiest 98 %.  With a top-k it is the three barriers (the first arrived at early) and
// the dependent passes between them that are left over the logits' read.
// Measured: a row of 128 256 f32 logits with top-k 40 and top-p 0.95 in 10.5 us, 64 such rows in 32 us; 200 rows of 32 000 bf16 logits with top-p alone in 67 us.
#pragma once
#include <cfloat>

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
    const float *temperature, *top_p, *min_p;  // of each row; null: the same for all, as below
    const int* top_k;
    const double* uniform;
    float same_temperature, same_top_p, same_min_p;
    int same_top_k;
    double same_uniform;
    int* tokens;
    float* probs;  // may be null
};

struct SampleShared {
    union {
        struct {
            uint32_t low[FS_BINS], high[FS_BINS];  // of each bin: the count in `low`, or the mass
        };
        uint64_t w[FS_LIST];  // masses of `all`, once all blocks have read the bins (a gathering's barrier is behind that)
    };
    uint64_t all[FS_LIST];     // keys that the blocks have listed
    uint64_t sorted[FS_FAST];
    double table[FS_TABLE];    // 2^(-i / FS_TABLE)
    uint64_t sums[FS_WARPS];
    float wmax[FS_WARPS], wmin[FS_WARPS], tmax[FS_THREADS];
    float queue[FS_WARPS][160];
    // of each block of the cluster, written by it
    float max[FS_CLUSTER], min[FS_CLUSTER], tau[FS_CLUSTER];
    uint32_t count[3][FS_CLUSTER];  // listed for a top-k, for the bin with the k-th value, for the nucleus' bin
    uint64_t total[3][FS_CLUSTER];  // two in turn, and the last one
    uint32_t listed[3];             // of the first block: where the next keys go
    // found by one thread, used by all
    float own_tau;
    uint32_t survivors, base;
    int bin;
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
    double dtop, rate;  // w = 2^-t, t = (top - x) * rate
    double min_p;       // at most 1: the first token is always kept
    const double* table;
    bool infinite;      // top
    // 2^-t: t to the nearest 1/128 from the table, the rest by the exponential series up to its fourth power (|rest * ln 2| <= 0.0027, whose fifth over 120 is
    // 1.2e-15).  No branch: beyond 100 (of -inf, too) t is 100, and the mass 0.
    __device__ __forceinline__ double weight(float x) const {
        if (infinite) return x == top ? 1.0 : 0.0;
        double t = (dtop - (double)x) * rate;
        t = t < 100.0 ? t : 100.0;
        constexpr double magic = 6755399441055744.0 / FS_TABLE, l = 0.6931471805599453;  // 1.5 * 2^52 / 128: the sum's last bit is 1/128
        const double u = t + magic;
        const int k = __double2loint(u);
        const double rest = t - (u - magic), q = fma(rest, fma(rest, fma(rest, fma(rest, l * l * l * l / 24, -l * l * l / 6), l * l / 2), -l), 1.0) * table[k & (FS_TABLE - 1)];
        return __hiloint2double(__double2hiint(q) - (k / FS_TABLE << 20), __double2loint(q));
    }
    // In units of 2^-44, to the nearest: the last bits of w + 2^8.
    static __device__ __forceinline__ uint64_t units(double w) {
        const double v = w + 256.0;
        return (uint64_t)(uint32_t)(__double2hiint(v) - 0x40700000) << 32 | (uint32_t)__double2loint(v);
    }
    __device__ __forceinline__ uint64_t mass(float x) const { return units(weight(x)); }
    // of a value that the order keeps
    __device__ __forceinline__ uint64_t kept_mass(float x) const {
        const double w = weight(x);
        return w >= min_p ? units(w) : 0;
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

// How many of the first n of `keys` are above keys[i], for each i: several threads share an i when there are few, and one of them calls body(i, count).
template <class Body>
__device__ __forceinline__ void places(const uint64_t* keys, int n, Body&& body) {
    int lanes = 16;
    while (lanes > 1 && FS_THREADS / lanes < n) lanes /= 2;
    const int q = threadIdx.x % lanes;
    for (int i0 = 0; i0 < n; i0 += FS_THREADS / lanes) {  // (the same for all threads)
        const int i = i0 + (int)threadIdx.x / lanes;
        const uint64_t key = i < n ? keys[i] : ~0ull;
        uint32_t place = 0;
#pragma unroll 8
        for (int j = q; j < n; j += lanes) place += keys[j] > key;
        for (int o = 1; o < lanes; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
        if (q == 0 && i < n) body(i, place);
    }
}
// The same with the mass above: of keys[j], mass[j].
template <class Body>
__device__ __forceinline__ void masses_above(const uint64_t* keys, const uint64_t* mass, int n, Body&& body) {
    int lanes = 16;
    while (lanes > 1 && FS_THREADS / lanes < n) lanes /= 2;
    const int q = threadIdx.x % lanes;
    for (int i0 = 0; i0 < n; i0 += FS_THREADS / lanes) {
        const int i = i0 + (int)threadIdx.x / lanes;
        const uint64_t key = i < n ? keys[i] : ~0ull;
        uint64_t above = 0;
#pragma unroll 4
        for (int j = q; j < n; j += lanes) above += keys[j] > key ? mass[j] : 0;
        for (int o = 1; o < lanes; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
        if (q == 0 && i < n) body(i, above);
    }
}

template <typename T>
__global__ void __launch_bounds__(FS_THREADS, 2) filtered_sample_kernel(const __grid_constant__ SampleParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) float fs_x[];
    __shared__ SampleShared s;
    const cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)blockIdx.x % p.cluster, row = (int)(blockIdx.x / p.cluster);
    const int first = rank * p.slice, n = max(0, min(p.slice, p.vocab - first)), quads = (n + 3) / 4;
    if (tid < FS_TABLE) s.table[tid] = exp2(-(double)tid / FS_TABLE);
    for (int i = tid; i < FS_BINS; i += FS_THREADS) s.low[i] = s.high[i] = 0;
    if (tid < 3) s.listed[tid] = 0;
    if (tid == 0) {
        s.survivors = 0;
        s.own_tau = -INFINITY;
    }
    cluster_arrive();  // (waited for before the first word goes to another block: that block has begun, and its counters are zero)
    pdl_wait();
    const float temperature = p.temperature ? p.temperature[row] : p.same_temperature;
    const int k = p.top_k ? p.top_k[row] : p.same_top_k;
    const float top_p = p.top_p ? p.top_p[row] : p.same_top_p, min_p = p.min_p ? p.min_p[row] : p.same_min_p;
    double u = p.uniform ? p.uniform[row] : p.same_uniform;

    // the slice, its maximum and its smallest finite value; no numbers become -inf, which is no choice
    float mx = -INFINITY, mn = INFINITY;
    auto take = [&](float x) {
        x = fmaxf(x, -INFINITY);
        mx = fmaxf(mx, x);
        mn = fminf(mn, x > -INFINITY ? x : INFINITY);
        return x;
    };
    const T* const src = (const T*)p.logits + row * p.stride + first;
    constexpr int V = 16 / sizeof(T);
    const int nv = ((uintptr_t)src & 15) == 0 ? n / V : 0;
#pragma unroll 4
    for (int i = tid; i < nv; i += FS_THREADS) {
        float x[V];
        get(src + i * V, x);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = take(x[e]);
#pragma unroll
        for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(fs_x + i * V + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
    }
#pragma unroll 8
    for (int i = nv * V + tid; i < n; i += FS_THREADS) fs_x[i] = take(to_f32(src[i]));
    if (tid < quads * 4 - n) fs_x[n + tid] = -INFINITY;
    const float own_max = mx;
    mx = warp_max(mx);
    mn = -warp_max(-mn);
    // The block's share of the k-th place: the value at that place among its threads' maxima.  Only those count that are as large as the weakest warp's
    // value at its own share of that place: there are enough of them.
    const bool fast = k > 1 && k <= FS_FAST;
    const int place = fast ? (k + p.cluster - 1) / p.cluster - 1 : 0;
    float mine = mx;
    if (fast) {
        float left = own_max;
        for (int j = place / FS_WARPS; j > 0; --j) {  // the warp's largest maxima one after the other
            const unsigned with = __ballot_sync(0xffffffffu, left == mine);
            if (lane == __ffs(with) - 1) left = -INFINITY;
            mine = warp_max(left);
        }
    }
    if (lane == 0) {
        s.wmax[warp] = mx;
        s.wmin[warp] = mn;
        s.sums[warp] = __float_as_uint(mine);
    }
    __syncthreads();
    float weakest = INFINITY;
    mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < FS_WARPS; ++w) {
        mx = fmaxf(mx, s.wmax[w]);
        mn = fminf(mn, s.wmin[w]);
        weakest = fminf(weakest, __uint_as_float((uint32_t)s.sums[w]));
    }
    if (fast) {
        const bool in = own_max >= weakest;
        const unsigned v = __ballot_sync(0xffffffffu, in);
        uint32_t at = 0;
        if (lane == 0 && v) at = atomicAdd(&s.survivors, __popc(v));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(v & ((1u << lane) - 1u));
        if (in) s.tmax[at] = own_max;
        __syncthreads();
        const int m = (int)s.survivors;
        if (tid < m) {
            const float t = s.tmax[tid];
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < m; ++j) above += s.tmax[j] > t || (s.tmax[j] == t && j < tid);
            if (above == place) s.own_tau = t;
        }
        __syncthreads();
    }
    cluster_wait();
    if (tid < p.cluster) {
        SampleShared* const o = cluster.map_shared_rank(&s, tid);
        o->max[rank] = mx;
        o->min[rank] = mn;
        o->tau[rank] = s.own_tau;
    }
    cluster.sync();
    float tau = INFINITY;
    for (int b = 0; b < p.cluster; ++b) {
        mx = fmaxf(mx, s.max[b]);
        mn = fminf(mn, s.min[b]);
        tau = fminf(tau, s.tau[b]);
    }
    const bool has_p = top_p < 1.f;
    if (mx == -INFINITY || !(temperature > 0.f) || k == 1 || top_p <= 0.f) {  // nothing to choose from, or to choose: the first maximum
        int b = 0;
        while (s.max[b] < mx) ++b;
        if (rank != b) return;
        if (tid == 0) s.base = 0xffffffffu;
        __syncthreads();
        for (int i = tid; i < n; i += FS_THREADS)
            if (fs_x[i] == mx) {
                atomicMin(&s.base, (uint32_t)(first + i));
                break;
            }
        __syncthreads();
        if (tid == 0) {
            p.tokens[row] = mx > -INFINITY ? (int)s.base : -1;
            if (p.probs) p.probs[row] = mx > -INFINITY ? 1.f : 0.f;
        }
        return;
    }
    SampleRow r;
    r.top = mx;
    r.infinite = mx == INFINITY;
    r.dtop = (double)mx;
    r.rate = 1.4426950408889634 / (double)temperature;
    r.min_p = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;
    r.table = s.table;
    u = u > 0.0 ? fmin(u, 1.0) : 0.0;
    // the last of the mass counts as not reached: u * whole rounds to at most whole, and the token is there where the sum exceeds it
    auto border = [&](uint64_t whole) { return min((uint64_t)(u * (double)whole), whole - 1); };
    const float span = fminf(mx - mn, 32.f * temperature);
    const float per = span > 1e-30f ? (float)FS_BINS / span : 1e30f;  // (an infinite span: everything in bin 0)
    auto bin_of = [&](float x) { return min(FS_BINS - 1, (int)((mx - x) * per)); };
    uint64_t cut = 0;  // key of the last that is kept

    // Values between lo and hi that pass `wanted`, of all blocks, to the first block's list or to everyone's.  Returns how many there are; more than FS_LIST:
    // no list.  One barrier of the cluster.
    auto gather = [&](int which, bool everyone, float lo, float hi, auto&& wanted) -> uint32_t {
        uint32_t mine = 0;
        for (int i = tid; i < quads; i += FS_THREADS) {
            const float4 x = *reinterpret_cast<const float4*>(fs_x + 4 * i);
            const float xs[4] = {x.x, x.y, x.z, x.w};
            if ((xs[0] >= lo && xs[0] <= hi) || (xs[1] >= lo && xs[1] <= hi) || (xs[2] >= lo && xs[2] <= hi) || (xs[3] >= lo && xs[3] <= hi)) {
                for (int e = 0; e < 4; ++e) mine += xs[e] >= lo && xs[e] <= hi && wanted(xs[e], order_key(xs[e], (uint32_t)(first + 4 * i + e)));
            }
        }
        uint32_t at = (uint32_t)block_before(mine, s);
        if (tid == FS_THREADS - 1) {
            const uint32_t here = at + mine;
            s.base = here && here <= FS_LIST ? atomicAdd(&cluster.map_shared_rank(&s, 0)->listed[which], here) : FS_LIST;
            for (int b = 0; b < p.cluster; ++b) cluster.map_shared_rank(&s, b)->count[which][rank] = here;
        }
        __syncthreads();
        at += s.base;
        if (mine) {
            for (int i = tid; i < quads; i += FS_THREADS) {
                const float4 q = *reinterpret_cast<const float4*>(fs_x + 4 * i);
                if (!((q.x >= lo && q.x <= hi) || (q.y >= lo && q.y <= hi) || (q.z >= lo && q.z <= hi) || (q.w >= lo && q.w <= hi))) continue;
                for (int e = 0; e < 4; ++e) {
                    const float x = fs_x[4 * i + e];
                    const uint64_t key = order_key(x, (uint32_t)(first + 4 * i + e));
                    if (x >= lo && x <= hi && wanted(x, key)) {
                        if (at < FS_LIST)
                            for (int b = 0; b < (everyone ? p.cluster : 1); ++b) cluster.map_shared_rank(&s, b)->all[at] = key;
                        ++at;
                    }
                }
            }
        }
        cluster.sync();
        uint32_t all = 0;
        for (int b = 0; b < p.cluster; ++b) all += min(s.count[which][b], (uint32_t)FS_LIST + 1);
        return all;
    };
    // where the values of a bin lie, with room for the rounding of both ways to say it; -inf is in none
    auto bin_low = [&](int b) { return b == FS_BINS - 1 ? -FLT_MAX : fmaxf(-FLT_MAX, mx - ((float)b + 1.02f) / per - fabsf(mx) * 0x1p-21f); };
    auto bin_high = [&](int b) { return b == 0 ? INFINITY : mx - ((float)b - 0.02f) / per + fabsf(mx) * 0x1p-21f; };
    // The smallest key c with measure(keys above c) below `most`: what is kept is c and all above it.  A pass over the row per bit.
    auto bisect = [&](auto&& measure, double most) -> uint64_t {
        uint64_t lo = (uint64_t)ordered_bits(mn) << 32, hi = order_key(mx, 0);  // holds at hi: nothing is above it
        int turn = 0;
        while (lo < hi) {
            const uint64_t mid = lo + (hi - lo) / 2;
            uint64_t v = 0;
            for (int i = tid; i < n; i += FS_THREADS) {
                const uint64_t key = order_key(fs_x[i], (uint32_t)(first + i));
                if (fs_x[i] > -INFINITY && key > mid) v += measure(fs_x[i], key);
            }
            v = block_total(v, s);
            if (tid < p.cluster) cluster.map_shared_rank(&s, tid)->total[turn][rank] = v;
            cluster.sync();
            uint64_t all = 0;
            for (int b = 0; b < p.cluster; ++b) all += s.total[turn][b];
            turn ^= 1;  // (the other slot: a block may be a step ahead)
            if ((double)all < most) hi = mid;
            else lo = mid + 1;
        }
        cluster.sync();
        return lo;
    };
    // The bin at which the running measure (counts, or masses) reaches `most`, and the measure before it and with it; the last bin, which is not measured, has the rest.
    auto reach = [&](double most, bool masses) {
        uint64_t c[FS_BINS / FS_THREADS], sum = 0;
#pragma unroll
        for (int e = 0; e < FS_BINS / FS_THREADS; ++e) c[e] = 0;
#pragma unroll 4
        for (int b = 0; b < p.cluster; ++b) {
            const SampleShared* o = cluster.map_shared_rank(&s, b);
            const uint2 low = *reinterpret_cast<const uint2*>(&o->low[2 * tid]);
            c[0] += low.x;
            c[1] += low.y;
            if (masses) {
                const uint2 high = *reinterpret_cast<const uint2*>(&o->high[2 * tid]);
                c[0] += (uint64_t)high.x << 32;
                c[1] += (uint64_t)high.y << 32;
            }
        }
        sum = c[0] + c[1];
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
    static_assert(FS_BINS == 2 * FS_THREADS && FS_FAST <= FS_THREADS, "two bins, or one kept value, to a thread");

    if (k > 0 && k < p.vocab) {
        uint32_t m = FS_LIST + 1;
        if (fast) m = gather(0, false, fmaxf(tau, -FLT_MAX), INFINITY, [](float, uint64_t) { return true; });
        if (m <= FS_LIST) {
            // everything that is kept is among these
            if (rank != 0) return;
            const int most_k = min(k, (int)m);
            places(s.all, (int)m, [&](int i, uint32_t at) {
                if (at < (uint32_t)most_k) s.sorted[at] = s.all[i];
            });
            __syncthreads();
            // a kept value to a thread, in order
            const uint64_t key = tid < most_k ? s.sorted[tid] : 0;
            uint64_t w = tid < most_k ? r.mass(from_ordered((uint32_t)(key >> 32))) : 0;
            if (has_p) {
                const uint64_t above = block_before(w, s);
                const double most = (double)top_p * (double)block_total(w, s);
                if (!((double)above < most) && tid > 0) w = 0;
            }
            if (w) w = r.kept_mass(from_ordered((uint32_t)(key >> 32)));
            if (tid < most_k) {
                s.all[tid] = key & 0xffffffffu;  // by index: the lower, the higher
                s.w[tid] = w;
            }
            const uint64_t whole = block_total(w, s), most_u = border(whole);  // (with barriers)
            masses_above(s.all, s.w, most_k, [&](int i, uint64_t above) {
                if (above <= most_u && most_u < above + s.w[i]) {  // (of one value only)
                    p.tokens[row] = (int)(0xffffffffu - (uint32_t)s.all[i]);
                    if (p.probs) p.probs[row] = (float)((double)s.w[i] / (double)whole);
                }
            });
            return;
        }
        uint32_t usable = 0;
        for (int i = tid; i < n; i += FS_THREADS) {
            const float x = fs_x[i];
            const int b = x > -INFINITY ? bin_of(x) : FS_BINS - 1;
            usable += x > -INFINITY;
            if (b < FS_BINS - 1) atomicAdd(&s.low[b], 1u);
        }
        usable = (uint32_t)block_total(usable, s);
        if (tid < p.cluster) cluster.map_shared_rank(&s, tid)->total[2][rank] = usable;
        cluster.sync();
        usable = 0;
        for (int b = 0; b < p.cluster; ++b) usable += (uint32_t)s.total[2][b];
        if ((uint32_t)k < usable) {
            reach((double)k, false);
            const int bk = s.bin;
            const uint32_t ahead = (uint32_t)s.before, upto = s.found != ~0ull ? (uint32_t)s.found : usable;
            if (upto - ahead <= FS_LIST) {
                m = gather(1, true, bin_low(bk), bin_high(bk), [&](float x, uint64_t) { return bin_of(x) == bk; });
                places(s.all, (int)m, [&](int i, uint32_t at) {
                    if (ahead + at == (uint32_t)k - 1) s.found = s.all[i];
                });
                __syncthreads();
                cut = s.found;
            } else {
                cut = bisect([](float, uint64_t) { return (uint64_t)1; }, (double)k);
            }
        }
        if (has_p) {
            cluster.sync();  // (all have read the counts)
            for (int i = tid; i < FS_BINS; i += FS_THREADS) s.low[i] = s.high[i] = 0;
            __syncthreads();
        }
    }

    if (has_p) {
        uint64_t sum = 0;
#pragma unroll 1
        for (int i = tid; i < quads; i += FS_THREADS) {
            const float4 x4 = *reinterpret_cast<const float4*>(fs_x + 4 * i);
            const float x[4] = {x4.x, x4.y, x4.z, x4.w};
            uint64_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = r.mass(x[e]);  // (of -inf: 0)
            if (cut != 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = order_key(x[e], (uint32_t)(first + 4 * i + e)) >= cut ? w[e] : 0;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum += w[e];
                const int b = bin_of(x[e]);
                if (w[e] && b < FS_BINS - 1) add_mass(s, b, w[e]);
            }
        }
        sum = block_total(sum, s);
        if (tid < p.cluster) cluster.map_shared_rank(&s, tid)->total[2][rank] = sum;
        cluster.sync();
        uint64_t whole = 0;
        for (int b = 0; b < p.cluster; ++b) whole += s.total[2][b];
        const double most = (double)top_p * (double)whole;
        reach(most, true);
        const int bp = s.bin;
        const uint64_t ahead = s.before;
        const uint32_t m = gather(2, true, bin_low(bp), bin_high(bp), [&](float x, uint64_t key) { return bin_of(x) == bp && key >= cut; });
        if (m <= FS_LIST) {
            for (uint32_t i = tid; i < m; i += FS_THREADS) s.w[i] = r.mass(from_ordered((uint32_t)(s.all[i] >> 32)));
            if (tid == 0) s.found = order_key(mx, 0);
            __syncthreads();
            masses_above(s.all, s.w, (int)m, [&](int i, uint64_t above) {  // (the first of a row has nothing before it, and it is less than most)
                if ((double)(ahead + above) < most) atomicMin((unsigned long long*)&s.found, (unsigned long long)s.all[i]);
            });
            __syncthreads();
            cut = max(cut, s.found);
        } else {
            const uint64_t old = cut;
            cut = max(old, bisect([&](float x, uint64_t key) { return key >= old ? r.mass(x) : (uint64_t)0; }, most));
        }
    }

    // the choice among all that is kept: masses per warp's stretch of the slice, then inside the stretch that holds it
    const double floor_t = r.min_p > 0.0 ? fmin(46.0, fmax(1e-6, 1e-6 - log2(r.min_p))) : 46.0;  // (a little beyond min_p: the comparison is made on the weight)
    const int stretch = ((p.slice + FS_WARPS - 1) / FS_WARPS + 127) / 128 * 128;
    // no smaller value is kept: the cut's, or the one from which on weights vanish (or are below min_p), with room for rounding
    const float low = fmaxf(fmaxf(from_ordered((uint32_t)(cut >> 32) | (cut ? 0u : 0x00800000u)), -FLT_MAX), mx - (float)(floor_t / r.rate) * 1.0001f - fabsf(mx) * 0x1p-21f);
    auto kept = [&](int i) -> uint64_t {
        const float x = fs_x[i];
        return x >= low && order_key(x, (uint32_t)(first + i)) >= cut ? r.kept_mass(x) : 0;
    };
    const int lo = min(n, warp * stretch), hi = min(n, lo + stretch);
    uint64_t sum = 0;
    int queued = 0;
    for (int i0 = lo; i0 < hi; i0 += 128) {
        const int i = i0 + 4 * lane;  // (what lies behind the slice's end up to a multiple of 4 is -inf)
        float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (i < hi) q = *reinterpret_cast<const float4*>(fs_x + i);
        const float x[4] = {q.x, q.y, q.z, q.w};
        bool in[4];
        int mine = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            in[e] = x[e] >= low && (x[e] > low || order_key(x[e], (uint32_t)(first + i + e)) >= cut);
            mine += in[e];
        }
        if (__all_sync(0xffffffffu, mine >= 2)) {  // (most of them: as they lie)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += in[e] ? r.kept_mass(x[e]) : 0;
            continue;
        }
        int at = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += v;
        }
        const int all = __shfl_sync(0xffffffffu, at, 31);
        at += queued - mine;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (in[e]) s.queue[warp][at++] = x[e];
        queued += all;
        __syncwarp();
        while (queued >= 32) {  // the last ones
            queued -= 32;
            sum += r.kept_mass(s.queue[warp][queued + lane]);
        }
        __syncwarp();
    }
    if (lane < queued) sum += r.kept_mass(s.queue[warp][lane]);
    sum = warp_sum64(sum);
    __syncthreads();
    if (lane == 0) s.sums[warp] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < FS_WARPS; ++w) sum += s.sums[w];
    if (tid < p.cluster) cluster.map_shared_rank(&s, tid)->total[1][rank] = sum;
    cluster.sync();
    uint64_t whole = 0, ahead = 0;
    for (int b = 0; b < p.cluster; ++b) {
        whole += s.total[1][b];
        ahead += b < rank ? s.total[1][b] : 0;
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
}

}  // namespace l2b
