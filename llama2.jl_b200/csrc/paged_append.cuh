// New rows of queries, keys and values on their way into a paged cache, in one pass: rms norm of each query and key head,
//   y = x / sqrt(mean(x^2) + eps) * gain,
// rotation of the pairs (a, b) = (y_2i, y_2i+1) or (y_i, y_i+size/2) by t = position * base^(-2i / size),
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),
// queries to the caller's buffer, keys and values into their pages, rounded once.  Everything is read once and written once, so memory bounds it.
// A group of threads holds one head: each thread two pieces of P values, half a head apart, so that pairs that lie half a head apart are one thread's and
// so are adjacent ones, and the norm is a few shuffles.  A warp works on the heads of one token.  Gains, cosines and sines of a thread's values are the
// same for all of them and become four coefficients per pair once (a' = r (A a - B b), b' = r (C a + D b), r = 1 / sqrt(..)), in registers: norm and rotation
// cost three operations a value.  (With gains and angles applied one after the other, and a kind looked up for each head, the instructions took twice the
// memory's time.)  The angles of a token are shared by its heads: a block computes them once for its tokens, in 64 bits up to the fraction of a
// turn (a far position times the fastest frequency would lose all of a turn in 32).
// Measured: 12 000 rows of 64 + 16 heads of 128 bf16 values (491 MB) in 102 us, 4.8 TB/s, 0.74 of the copy rate; one row of 32 + 16 heads in 3.5 us, a launch and its look-ups.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "paged.h"

namespace l2b {

constexpr int PA_THREADS = 256, PA_MAX_SIZE = 128, PA_MAX_TOKENS = 8, PA_WARPS = PA_THREADS / 32;

struct AppendParams {
    PagedPool pool;
    PagedSeqs seqs;
    const void *q, *k, *v;  // q may be null
    void* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const float *q_gain, *k_gain;  // null: no norm
    float eps, inv_size;
    int n_heads, tokens;  // tokens of a block
    double turns[PA_MAX_SIZE / 2];      // turns per position
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N values of T at a place that is aligned to them, up to 16 bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void get(const T* p, float (&x)[N]) {
    const Pack<T, N> a = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(a.v[i]);
}
// N values as they were loaded, in words.
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Words {
    uint32_t w[sizeof(T) * N / 4];
    __device__ __forceinline__ float value(int i) const {
        if (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint32_t p = w[i / 2];
        if (std::is_same<T, __half>::value) return half_bits_to_float(i & 1 ? p >> 16 : p & 0xffffu);
        return __uint_as_float(i & 1 ? p & 0xffff0000u : p << 16);
    }
};
template <typename T, int N>
__device__ __forceinline__ void put(T* p, const float (&x)[N]) {
    Pack<T, N> a;
#pragma unroll
    for (int i = 0; i < N; ++i) a.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Pack<T, N>*>(p) = a;
}

// What rotation pairs.  Without it no pairs are formed at all: with sines of 0 an infinite value would be no number in its partner's place.
enum RowPairs { PAIRS_NONE, PAIRS_NEIGHBOURS, PAIRS_HALF_APART };

// TI: type of the rows, TC: of the cache, P: values of a piece (8, or 4 for heads that are no multiple of 16)
template <typename TI, typename TC, int P, RowPairs PAIRS>
__global__ void __launch_bounds__(PA_THREADS, 3) paged_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int AHEAD = 32 / (P * (int)sizeof(TI));  // groups of heads under way
    constexpr bool ROTATE = PAIRS != PAIRS_NONE, NEOX = PAIRS == PAIRS_HALF_APART;
    __shared__ __align__(16) float2 s_cs[PA_MAX_TOKENS][PA_MAX_SIZE / 2];
    __shared__ int s_page[PA_MAX_TOKENS], s_slot[PA_MAX_TOKENS], s_new[PA_MAX_TOKENS];
    const int hs = p.pool.hs, half = hs / 2, units = hs / (2 * P), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int lanes = 1;
    while (lanes < units) lanes *= 2;
    const int unit = lane % lanes, at_once = 32 / lanes;  // heads of a warp at once
    const bool active = unit < units;
    // where this thread's two pieces lie in a head
    const int d0 = unit * P, d1 = half + d0;
    const int nq = p.q ? p.n_heads : 0, q_groups = (nq + at_once - 1) / at_once, kv_groups = (p.pool.n_kv + at_once - 1) / at_once;
    const int64_t rows = (int64_t)p.seqs.n_seq * p.seqs.n_query, row0 = (int64_t)blockIdx.x * p.tokens;
    const int here = (int)(rows - row0 < p.tokens ? rows - row0 : p.tokens);
    pdl_wait();

    if (tid < here) {
        const int64_t row = row0 + tid;
        const int seq = (int)(row / p.seqs.n_query), j = (int)(row - (int64_t)seq * p.seqs.n_query);
        const int length = p.seqs.lengths[seq], count = paged_count(length, p.seqs.counts ? p.seqs.counts[seq] : p.seqs.n_query, p.seqs.n_query);
        const int pos = length - count + j;  // own position
        int page = -1;
        if (j < count && pos >= 0 && pos < paged_keys(length, p.seqs.width, p.pool.page_shift))
            page = p.seqs.pages[(int64_t)seq * p.seqs.width + (pos >> p.pool.page_shift)];
        s_page[tid] = page >= 0 && page < p.pool.n_pages ? page : -1;
        s_slot[tid] = pos & ((1 << p.pool.page_shift) - 1);
        s_new[tid] = j < count;
    }
    if constexpr (ROTATE) {
        for (int i = tid; i < here * half; i += PA_THREADS) {
            const int t = i / half, f = i - t * half;
            const int64_t row = row0 + t;
            const int seq = (int)(row / p.seqs.n_query), j = (int)(row - (int64_t)seq * p.seqs.n_query);
            const int length = p.seqs.lengths[seq], count = paged_count(length, p.seqs.counts ? p.seqs.counts[seq] : p.seqs.n_query, p.seqs.n_query);
            const double turn = (double)((int64_t)p.seqs.prefix_len + length - count + j) * p.turns[f];
            float s, c;
            sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
            s_cs[t][f] = make_float2(c, s);
        }
    }
    __syncthreads();

    const int per_token = PA_WARPS / p.tokens, t = warp / per_token;  // warps of a token; this warp's
    if (t >= here || !s_new[t]) return;
    const int64_t row = row0 + t;
    const int page = s_page[t], stride = (int)gridDim.y * per_token, start = (int)blockIdx.y * per_token + warp % per_token, sub = lane / lanes;
    // Groups of heads kind by kind, one to each warp of the token in turn.  `of`: groups of the kinds before.
    auto heads = [&](auto kind, int n_heads, int n_groups, int of, const TI* src, auto* dst, int64_t dst_head, const float* gains) {
        constexpr bool VALUES = decltype(kind)::value;
        using TO = typename std::remove_pointer<decltype(dst)>::type;
        int g = start - of % stride;
        if (g < 0) g += stride;
        if (g >= n_groups) return;
        float ca[P], cb[P], cc[P], cd[P];  // of pairs (d0 + i, d1 + i), or of the adjacent ones of either piece
        if constexpr (!VALUES) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int da = NEOX ? d0 + i : (i < P / 2 ? d0 + 2 * i : d1 + 2 * i - P), db = NEOX ? d1 + i : da + 1;
                float2 cs = make_float2(1.f, 0.f);
                float ga = 1.f, gb = 1.f;
                if (ROTATE && active) cs = s_cs[t][NEOX ? da : da / 2];
                if (active && gains) {
                    ga = gains[da];
                    gb = gains[db];
                }
                ca[i] = ga * cs.x;
                cb[i] = gb * cs.y;
                cc[i] = ga * cs.y;
                cd[i] = gb * cs.x;
            }
        }
        for (; g < n_groups; g += AHEAD * stride) {
            Words<TI, P> raw[AHEAD][2];
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) {
                const int h = (g + n * stride) * at_once + sub;
                if (active && h < n_heads) {
                    const TI* const from = src + (int64_t)h * hs;
                    raw[n][0] = *reinterpret_cast<const Words<TI, P>*>(from + d0);
                    raw[n][1] = *reinterpret_cast<const Words<TI, P>*>(from + d1);
                }
            }
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) {
                const int h = (g + n * stride) * at_once + sub;
                const bool go = active && h < n_heads;
                float x[2][P], r = 1.f;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    x[0][i] = go ? raw[n][0].value(i) : 0.f;
                    x[1][i] = go ? raw[n][1].value(i) : 0.f;
                }
                if constexpr (!VALUES) {
                    if (gains) {
                        float ss = 0.f;
#pragma unroll
                        for (int i = 0; i < P; ++i) ss = fmaf(x[0][i], x[0][i], fmaf(x[1][i], x[1][i], ss));
                        for (int o = lanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                        r = rsqrtf(fmaf(ss, p.inv_size, p.eps));
                    }
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        float& xa = NEOX ? x[0][i] : x[2 * i / P][2 * i % P];
                        float& xb = NEOX ? x[1][i] : x[2 * i / P][2 * i % P + 1];
                        const float a = xa * r, b = xb * r;
                        xa = ROTATE ? a * ca[i] - b * cb[i] : a * ca[i];
                        xb = ROTATE ? a * cc[i] + b * cd[i] : b * cd[i];
                    }
                }
                if (go) {
                    TO* const to = dst + h * dst_head;
                    put(to + d0, x[0]);
                    put(to + d1, x[1]);
                }
            }
        }
    };
    if (nq) heads(std::false_type(), nq, q_groups, 0, (const TI*)p.q + row * p.q_stride, (TI*)p.q_out + row * p.q_out_stride, hs, p.q_gain);
    if (page >= 0) {
        const int64_t at = paged_offset(page, 0, s_slot[t], p.pool), head = (int64_t)hs << p.pool.page_shift;
        heads(std::false_type(), p.pool.n_kv, kv_groups, q_groups, (const TI*)p.k + row * p.k_stride, (TC*)p.pool.k + at, head, p.k_gain);
        heads(std::true_type(), p.pool.n_kv, kv_groups, q_groups + kv_groups, (const TI*)p.v + row * p.v_stride, (TC*)p.pool.v + at, head, nullptr);
    }
}

}  // namespace l2b
