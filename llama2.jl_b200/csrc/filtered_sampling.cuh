// The next token of each row of logits by temperature, top-k, top-p and min-p from a given random number.
//   w_i = exp((x_i - max) / T);  order: larger x first, of equal ones the lower index first.
//   top-k keeps the first k;  top-p keeps those before which less than p of the mass of what top-k keeps lies;  min-p keeps w_i >= min_p;  the first
//   is always kept.  The token is the first, by index, at which the kept tokens' cumulated mass exceeds u times their whole.
//
// A cluster of up to eight blocks holds a row in its shared memory, read once; every pass after that is over shared memory.  Masses are whole numbers of
// 2^-44 of the largest weight (weights computed in 64 bits), so that sums do not depend on their order and no cut or choice hangs on the blocks or on atomics.
// Cuts: equal bins of the distance from the maximum are counted; only the bin that holds the k-th value (or the nucleus' border) is ordered,
// by counting, a thread per value.  With a top-k whose bins hold at most LIST values everything else happens among those.  The nucleus' bin is first guessed from
// f32 masses per bin and then checked with exact sums.  More than LIST values in one bin (many equal logits): bisection on (value, index), a pass per bit.
// Bound by the passes over shared memory and by the cluster's barriers; the logits' read is the floor.
#pragma once
#include <cooperative_groups.h>

#include "paged_append.cuh"

namespace l2b {

constexpr int FS_THREADS = 512, FS_WARPS = FS_THREADS / 32, FS_BINS = 1024, FS_LIST = 1024, FS_CLUSTER = 8;
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
    uint32_t count[FS_BINS];
    float mass[FS_BINS];
    uint64_t list[FS_LIST];
    uint64_t all[FS_LIST], w[FS_LIST];  // block 0: the lists of all blocks, and their weights
    uint64_t sums[FS_WARPS];
    float wmax[FS_WARPS], wmin[FS_WARPS];
    uint32_t widx[FS_WARPS], wcnt[FS_WARPS];
    // what other blocks read
    float max, min;
    uint32_t idx, usable, listed;
    uint64_t total[2];
    uint64_t cut;
    // found by one thread, used by all
    int bin;
    uint32_t before;
    uint32_t choice;
    uint64_t found;
};

__device__ __forceinline__ uint32_t ordered_bits(float x) {  // larger value, larger number; -0 and 0 are equal
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) { return (uint64_t)ordered_bits(x) << 32 | (0xffffffffu - index); }

struct SampleRow {
    float max;
    double dmax, rate, floor_t;  // w = 2^-((max - x) * rate); floor_t: no weight beyond
    double min_p;
    uint64_t first;  // key of the first token: always kept
    __device__ __forceinline__ double weight(float x) const {
        if (x == max) return 1.0;
        const double t = (dmax - (double)x) * rate;
        return t < floor_t ? exp2(-t) : 0.0;  // (NaN: infinite minus infinite)
    }
    // mass of a value that the order keeps
    __device__ __forceinline__ uint64_t mass(float x) const {
        const double w = weight(x);
        return (uint64_t)__double2ll_rn(w * FS_ONE);
    }
    __device__ __forceinline__ uint64_t kept_mass(float x, uint64_t key) const {
        const double w = weight(x);
        return w >= min_p || key == first ? (uint64_t)__double2ll_rn(w * FS_ONE) : 0;
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

template <typename T>
__global__ void __launch_bounds__(FS_THREADS) filtered_sample_kernel(const __grid_constant__ SampleParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) float fs_x[];
    __shared__ SampleShared s;
    const cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)blockIdx.x % p.cluster, row = (int)(blockIdx.x / p.cluster);
    const int first = rank * p.slice, n = max(0, min(p.slice, p.vocab - first));
    pdl_wait();

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
    for (int i = tid; i < nv; i += FS_THREADS) {
        float x[V];
        get(src + i * V, x);
#pragma unroll
        for (int e = 0; e < V; ++e) take(i * V + e, x[e]);
    }
    for (int i = nv * V + tid; i < n; i += FS_THREADS) take(i, to_f32(src[i]));
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
    if (tid == 0) {
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
    }
    for (int i = tid; i < FS_BINS; i += FS_THREADS) {
        s.count[i] = 0;
        s.mass[i] = 0.f;
    }
    cluster.sync();
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
        usable += o->usable;
    }

    const float temperature = p.temperature ? p.temperature[row] : 1.f;
    const int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p && p.min_p[row] > 0.f ? p.min_p[row] : 0.f;
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
    r.max = mx;
    r.dmax = (double)mx;
    r.rate = 1.4426950408889634 / (double)temperature;
    r.floor_t = 46.0;
    r.min_p = (double)min_p;
    r.first = order_key(mx, mi);
    double u = p.uniform[row];
    u = u > 0.0 ? fmin(u, 1.0) : 0.0;
    // the last of the mass counts as not reached: u * whole rounds to at most whole, and the token is there where the sum exceeds it
    auto border = [&](uint64_t whole) { return min((uint64_t)(u * (double)whole), whole - 1); };

    const float span = fminf(mx - mn, 32.f * temperature);
    const float per = span > 1e-30f ? (float)FS_BINS / span : 1e30f;  // (an infinite span: everything in bin 0)
    auto bin_of = [&](float x) { return min(FS_BINS - 1, (int)((mx - x) * per)); };
    uint64_t cut = 0;  // key of the last that is kept

    // Values of one kind, listed by every block, brought together by block 0.  Returns how many there are (all blocks know; more than FS_LIST: no list).
    auto gather = [&](auto&& wanted) -> uint32_t {
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
        uint32_t all = 0, mine = 0;
        for (int b = 0; b < p.cluster; ++b) all += cluster.map_shared_rank(&s, b)->listed;
        if (rank == 0 && all <= FS_LIST) {
            for (int b = 0; b < p.cluster; ++b) {
                const SampleShared* o = cluster.map_shared_rank(&s, b);
                const uint32_t c = o->listed;
                for (uint32_t i = tid; i < c; i += FS_THREADS) {
                    const uint64_t key = o->list[i];
                    s.all[mine + i] = key;
                    s.w[mine + i] = r.mass(from_ordered((uint32_t)(key >> 32)));
                }
                mine += c;
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

    bool chosen = false;
    if (has_k) {
        for (int i = tid; i < n; i += FS_THREADS) {
            const int b = fs_x[i] > -INFINITY ? bin_of(fs_x[i]) : FS_BINS - 1;
            if (b < FS_BINS - 1) atomicAdd(&s.count[b], 1u);  // (the last bin has the rest)
        }
        if (tid == 0) {
            s.bin = FS_BINS - 1;
            s.before = 0xffffffffu;
        }
        cluster.sync();
        uint32_t c[FS_BINS / FS_THREADS], sum = 0;
#pragma unroll
        for (int e = 0; e < FS_BINS / FS_THREADS; ++e) {
            c[e] = 0;
            for (int b = 0; b < p.cluster; ++b) c[e] += cluster.map_shared_rank(&s, b)->count[tid * (FS_BINS / FS_THREADS) + e];
            sum += c[e];
        }
        uint32_t before = (uint32_t)block_before(sum, s);
        const uint32_t binned = (uint32_t)block_total(sum, s);
#pragma unroll
        for (int e = 0; e < FS_BINS / FS_THREADS; ++e) {
            if (before < (uint32_t)k && before + c[e] >= (uint32_t)k) {
                s.bin = tid * (FS_BINS / FS_THREADS) + e;
                s.before = before;
                s.found = before + c[e];
            }
            before += c[e];
        }
        __syncthreads();
        const int bk = s.bin;
        const uint32_t ahead = s.before != 0xffffffffu ? s.before : binned, upto = s.before != 0xffffffffu ? (uint32_t)s.found : usable;
        if (upto <= FS_LIST) {
            // everything that is kept is among these
            gather([&](float x, uint32_t) { return bin_of(x) <= bk; });
            if (rank == 0) {
                const int m = (int)upto;
                uint64_t key[FS_LIST / FS_THREADS], w[FS_LIST / FS_THREADS], above[FS_LIST / FS_THREADS] = {}, mass_k = 0;
                uint32_t place[FS_LIST / FS_THREADS] = {};
#pragma unroll
                for (int e = 0; e < FS_LIST / FS_THREADS; ++e) {
                    const int i = tid + e * FS_THREADS;
                    key[e] = i < m ? s.all[i] : 0;
                    w[e] = i < m ? s.w[i] : 0;
                }
                for (int j = 0; j < m; ++j) {
                    const uint64_t kj = s.all[j], wj = s.w[j];
#pragma unroll
                    for (int e = 0; e < FS_LIST / FS_THREADS; ++e) {
                        place[e] += kj > key[e];
                        above[e] += kj > key[e] ? wj : 0;
                    }
                }
#pragma unroll
                for (int e = 0; e < FS_LIST / FS_THREADS; ++e) mass_k += place[e] < (uint32_t)k ? w[e] : 0;
                mass_k = block_total(mass_k, s);
                const double most = (double)top_p * (double)mass_k;
                uint64_t whole = 0;
#pragma unroll
                for (int e = 0; e < FS_LIST / FS_THREADS; ++e) {
                    const int i = tid + e * FS_THREADS;
                    const bool keep = i < m && place[e] < (uint32_t)k && (!has_p || (double)above[e] < most || key[e] == r.first);
                    w[e] = keep ? r.kept_mass(from_ordered((uint32_t)(key[e] >> 32)), key[e]) : 0;
                    whole += w[e];
                }
                whole = block_total(whole, s);  // (its barriers: everyone has read s.w)
#pragma unroll
                for (int e = 0; e < FS_LIST / FS_THREADS; ++e)
                    if (tid + e * FS_THREADS < m) s.w[tid + e * FS_THREADS] = w[e];
                if (tid == 0) s.choice = 0xffffffffu;
                __syncthreads();
                const uint64_t most_u = border(whole);
                uint64_t run[FS_LIST / FS_THREADS] = {};  // mass up to this one, by index
                for (int j = 0; j < m; ++j) {
                    const uint32_t kj = (uint32_t)s.all[j];  // (the higher the lower the index)
                    const uint64_t wj = s.w[j];
#pragma unroll
                    for (int e = 0; e < FS_LIST / FS_THREADS; ++e) run[e] += kj >= (uint32_t)key[e] ? wj : 0;
                }
#pragma unroll
                for (int e = 0; e < FS_LIST / FS_THREADS; ++e)
                    if (w[e] && run[e] > most_u) atomicMin(&s.choice, 0xffffffffu - (uint32_t)key[e]);
                __syncthreads();
#pragma unroll
                for (int e = 0; e < FS_LIST / FS_THREADS; ++e)
                    if (w[e] && 0xffffffffu - (uint32_t)key[e] == s.choice) {
                        p.tokens[row] = (int)s.choice;
                        if (p.probs) p.probs[row] = (float)((double)w[e] / (double)whole);
                    }
            }
            chosen = true;
        } else if (upto - ahead <= FS_LIST) {
            gather([&](float x, uint32_t) { return bin_of(x) == bk; });
            if (rank == 0) {
                const int m = (int)(upto - ahead);
                for (int i = tid; i < m; i += FS_THREADS) {
                    uint32_t place = ahead;
                    for (int j = 0; j < m; ++j) place += s.all[j] > s.all[i];
                    if (place == (uint32_t)k - 1) s.cut = s.all[i];
                }
            }
            cluster.sync();
            cut = cluster.map_shared_rank(&s, 0)->cut;
        } else {
            cut = bisect([](float, uint64_t) { return (uint64_t)1; }, (double)k);
        }
    }
    if (chosen) {
        cluster.sync();
        return;
    }

    if (has_p) {
        uint64_t sum = 0;
        for (int i = tid; i < n; i += FS_THREADS) {
            const float x = fs_x[i];
            if (x > -INFINITY && order_key(x, (uint32_t)(first + i)) >= cut) {
                const uint64_t w = r.mass(x);
                const int b = bin_of(x);
                sum += w;
                if (b < FS_BINS - 1) atomicAdd(&s.mass[b], (float)w);  // (a guess: its rounding hangs on the order)
            }
        }
        sum = block_total(sum, s);
        if (tid == 0) {
            s.total[0] = sum;
            s.bin = FS_BINS - 1;
        }
        cluster.sync();
        uint64_t whole = 0;
        for (int b = 0; b < p.cluster; ++b) whole += cluster.map_shared_rank(&s, b)->total[0];
        const double most = (double)top_p * (double)whole;
        if (rank == 0) {  // the guess
            float c[FS_BINS / FS_THREADS];
            uint64_t mine = 0;
#pragma unroll
            for (int e = 0; e < FS_BINS / FS_THREADS; ++e) {
                c[e] = 0.f;
                for (int b = 0; b < p.cluster; ++b) c[e] += cluster.map_shared_rank(&s, b)->mass[tid * (FS_BINS / FS_THREADS) + e];
                mine += (uint64_t)c[e];
            }
            uint64_t before = block_before(mine, s);
#pragma unroll
            for (int e = 0; e < FS_BINS / FS_THREADS; ++e) {
                const uint64_t after = before + (uint64_t)c[e];
                if ((double)before < most && (double)after >= most) s.bin = tid * (FS_BINS / FS_THREADS) + e;
                before = after;
            }
        }
        cluster.sync();
        int bp = cluster.map_shared_rank(&s, 0)->bin;
        uint64_t ahead = 0;
        uint32_t listed;
        for (;;) {  // one way only: down while too much lies before the bin, up while too little lies before its end
            uint64_t before = 0, in = 0;
            listed = gather([&](float x, uint32_t index) {
                if (order_key(x, index) < cut) return false;
                const int b = bin_of(x);
                if (b > bp) return false;
                const uint64_t w = r.mass(x);
                before += b < bp ? w : 0;
                in += b == bp ? w : 0;
                return b == bp;
            });
            before = block_total(before, s);
            in = block_total(in, s);
            if (tid == 0) {
                s.total[0] = before;
                s.total[1] = in;
            }
            cluster.sync();
            before = in = 0;
            for (int b = 0; b < p.cluster; ++b) {
                before += cluster.map_shared_rank(&s, b)->total[0];
                in += cluster.map_shared_rank(&s, b)->total[1];
            }
            cluster.sync();  // (all have read before any writes again)
            ahead = before;
            if ((double)before >= most && bp > 0) --bp;
            else if ((double)(before + in) < most && bp < FS_BINS - 1) ++bp;
            else break;
        }
        if (listed <= FS_LIST) {
            if (rank == 0) {
                if (tid == 0) s.found = ~0ull;
                __syncthreads();
                for (uint32_t i = tid; i < listed; i += FS_THREADS) {
                    uint64_t above = ahead;
                    for (uint32_t j = 0; j < listed; ++j) above += s.all[j] > s.all[i] ? s.w[j] : 0;
                    if ((double)above < most) atomicMin((unsigned long long*)&s.found, (unsigned long long)s.all[i]);
                }
                __syncthreads();
                if (tid == 0) s.cut = min(s.found, r.first);  // (the first is always kept)
            }
            cluster.sync();
            cut = max(cut, cluster.map_shared_rank(&s, 0)->cut);
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
    if (tid == 0) s.total[0] = sum;
    cluster.sync();
    uint64_t whole = 0, ahead = 0;
    for (int b = 0; b < p.cluster; ++b) {
        const uint64_t t = cluster.map_shared_rank(&s, b)->total[0];
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
