// New rows of queries, keys and values on their way into a paged cache, in one pass: rms norm of each query and key head,
//   y = x / sqrt(mean(x^2) + eps) * gain,
// rotation of the pairs (a, b) = (y_2i, y_2i+1) or (y_i, y_i+size/2) by t = position * base^(-2i / size),
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),
// queries to the caller's buffer, keys and values into their pages, rounded once.  Everything is read once and written once, so memory bounds it.
// A group of LANES threads holds one head: each thread one unit of U values, as two pieces that are each other's partners when the pairs lie half a
// head apart.  So the norm is a few shuffles, the gains stay in registers, and all accesses are of 16 bytes (heads of 8, 24, 40 .. values: 8 bytes
// for 16-bit types).  The angles of a token are shared by its heads: a block computes them once for its tokens, in 64 bits up to the fraction of a
// turn (a far position times the fastest frequency would lose all of a turn in 32), and the first heads' values are on their way meanwhile.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "paged.h"

namespace l2b {

constexpr int PA_THREADS = 256, PA_MAX_SIZE = 128, PA_MAX_TOKENS = 8;

struct AppendParams {
    PagedPool pool;
    PagedSeqs seqs;
    const void *q, *k, *v;  // q may be null
    void* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const float *q_gain, *k_gain;  // null: no norm
    float eps;
    int n_heads, rotate, neox, tokens;  // tokens of a block
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
template <typename T, int N>
__device__ __forceinline__ void put(T* p, const float (&x)[N]) {
    Pack<T, N> a;
#pragma unroll
    for (int i = 0; i < N; ++i) a.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Pack<T, N>*>(p) = a;
}

// TI: type of the rows, TC: of the cache, U: values of a thread (16, or 8 for heads that are no multiple of 16)
template <typename TI, typename TC, int U>
__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int P = U / 2;  // values of a piece
    __shared__ float2 s_cs[PA_MAX_TOKENS][PA_MAX_SIZE / 2];
    __shared__ int s_page[PA_MAX_TOKENS], s_slot[PA_MAX_TOKENS], s_new[PA_MAX_TOKENS];
    const int hs = p.pool.hs, half = hs / 2, units = hs / U, tid = threadIdx.x;
    int lanes = 1;
    while (lanes < units) lanes *= 2;
    const int unit = tid % lanes, heads_at_once = PA_THREADS / lanes;
    const bool active = unit < units;
    // where this thread's two pieces lie in a head
    const int d0 = p.neox ? unit * P : unit * U, d1 = p.neox ? half + unit * P : d0 + P;
    const int nq = p.q ? p.n_heads : 0, slots = nq + 2 * p.pool.n_kv;
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
    if (p.rotate) {
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
    float gq[2][P], gk[2][P];
#pragma unroll
    for (int i = 0; i < P; ++i) gq[0][i] = gq[1][i] = gk[0][i] = gk[1][i] = 1.f;
    if (active && p.q_gain) get(p.q_gain + d0, gq[0]), get(p.q_gain + d1, gq[1]);
    if (active && p.k_gain) get(p.k_gain + d0, gk[0]), get(p.k_gain + d1, gk[1]);
    __syncthreads();

    const int total = here * slots;
    for (int base = (int)blockIdx.y * heads_at_once; base < total; base += (int)gridDim.y * heads_at_once) {  // (the same for all threads of a warp)
        const int it = base + tid / lanes;
        const bool mine = it < total;
        const int t = mine ? it / slots : 0, h = it - t * slots;
        const int64_t row = row0 + t;
        const bool is_q = h < nq, is_v = h >= nq + p.pool.n_kv, go = mine && active && s_new[t] && (is_q || s_page[t] >= 0);
        float x[2][P];
        if (go) {
            const TI* src = is_q ? (const TI*)p.q + row * p.q_stride + (int64_t)h * hs
                                 : is_v ? (const TI*)p.v + row * p.v_stride + (int64_t)(h - nq - p.pool.n_kv) * hs : (const TI*)p.k + row * p.k_stride + (int64_t)(h - nq) * hs;
            get(src + d0, x[0]);
            get(src + d1, x[1]);
        }
        const bool norm = is_q ? p.q_gain != nullptr : !is_v && p.k_gain != nullptr;
        if (p.q_gain || p.k_gain) {
            float ss = 0.f;
            if (go && norm) {
#pragma unroll
                for (int i = 0; i < P; ++i) ss = fmaf(x[0][i], x[0][i], fmaf(x[1][i], x[1][i], ss));
            }
            for (int o = lanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (norm) {
                const float r = rsqrtf(ss / (float)hs + p.eps);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    x[0][i] *= r * (is_q ? gq[0][i] : gk[0][i]);
                    x[1][i] *= r * (is_q ? gq[1][i] : gk[1][i]);
                }
            }
        }
        if (!go) continue;
        if (p.rotate && !is_v) {
            if (p.neox) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float2 cs = s_cs[t][d0 + i];
                    const float a = x[0][i], b = x[1][i];
                    x[0][i] = a * cs.x - b * cs.y;
                    x[1][i] = a * cs.y + b * cs.x;
                }
            } else {
#pragma unroll
                for (int i = 0; i < U; i += 2) {
                    const float2 cs = s_cs[t][(d0 + i) / 2];
                    float &ra = i < P ? x[0][i % P] : x[1][i % P], &rb = i < P ? x[0][i % P + 1] : x[1][i % P + 1];
                    const float a = ra, b = rb;
                    ra = a * cs.x - b * cs.y;
                    rb = a * cs.y + b * cs.x;
                }
            }
        }
        if (is_q) {
            TI* dst = (TI*)p.q_out + row * p.q_out_stride + (int64_t)h * hs;
            put(dst + d0, x[0]);
            put(dst + d1, x[1]);
        } else {
            TC* dst = (TC*)(is_v ? p.pool.v : p.pool.k) + paged_offset(s_page[t], is_v ? h - nq - p.pool.n_kv : h - nq, s_slot[t], p.pool);
            put(dst + d0, x[0]);
            put(dst + d1, x[1]);
        }
    }
}

}  // namespace l2b
