// Entry points of the paged cache (append, attention) and of filtered sampling: argument checks, choice of kernel, launches.
#include <atomic>
#include <cmath>

#include "filtered_sampling.cuh"
#include "host_common.h"
#include "paged_attention.cuh"
#include "paged_prefix.cuh"
#include "serving.h"

using namespace l2b;

namespace {

constexpr int MAX_DEVICES = 64;
constexpr float LOG2E = 1.4426950408889634f;  // the kernels' exponents count in powers of two
static_assert(SAMPLE_MAX_VOCAB == FS_CLUSTER * FS_SLICE, "what a cluster's shared memory holds");

// The device that a pointer's memory is on is the current one while this lives.
struct OnDeviceOf {
    int before = -1;
    int32_t enter(const void* ptr, const char* what) {
        int n = 0;
        if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
            (void)cudaGetLastError();
            return fail(L2B_ERR_NO_DEVICE, "no CUDA device is visible; this library has no CPU path");
        }
        cudaPointerAttributes a;
        const cudaError_t e = cudaPointerGetAttributes(&a, ptr);
        if (e != cudaSuccess || (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)) {
            (void)cudaGetLastError();
            return fail(L2B_ERR_BAD_ARG, std::string(what) + " is not device memory");
        }
        int now = 0;
        CU(cudaGetDevice(&now));
        if (now != a.device) {
            CU(cudaSetDevice(a.device));
            before = now;
        }
        device = a.device;
        return L2B_OK;
    }
    ~OnDeviceOf() {
        if (before >= 0) (void)cudaSetDevice(before);
    }
    int device = 0;
};

int32_t sm_count(int device, int* sms) {
    static std::atomic<int> known[MAX_DEVICES];
    if (device >= 0 && device < MAX_DEVICES && (*sms = known[device].load()) > 0) return L2B_OK;
    CU(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
    if (device >= 0 && device < MAX_DEVICES) known[device].store(*sms);
    return L2B_OK;
}

// A kernel may take all shared memory of an SM: said once per kernel and device.
template <auto Kernel>
int32_t allow_smem(int device) {
    static std::atomic<uint64_t> said{0};
    const uint64_t bit = device >= 0 && device < MAX_DEVICES ? 1ull << device : 0;
    if (bit && (said.load() & bit)) return L2B_OK;
    cudaFuncAttributes a;
    CU(cudaFuncGetAttributes(&a, Kernel));
    CU(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)a.sharedSizeBytes));
    said.fetch_or(bit);
    return L2B_OK;
}

bool aligned(const void* p, size_t to = 16) { return ((uintptr_t)p & (to - 1)) == 0; }
int type_bytes(int type) { return type == L2B_TYPE_F32 ? 4 : 2; }

int32_t check_cache(const l2b_paged_cache* c, PagedPool& pool) {
    if (!c || !c->dev_k || !c->dev_v) return fail(L2B_ERR_BAD_ARG, "null argument");
    if (c->type != L2B_TYPE_F16 && c->type != L2B_TYPE_BF16) return fail(L2B_ERR_UNSUPPORTED_TYPE, "a paged cache holds f16 or bf16 values");
    if (c->n_pages <= 0 || c->n_kv_heads <= 0 || c->n_kv_heads > 65535) return fail(L2B_ERR_BAD_ARG, "bad number of pages or key/value heads");
    if (c->page_size < 8 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return fail(L2B_ERR_BAD_ARG, "page_size must be a power of two, 8 to 1024");
    if (c->head_size < 8 || c->head_size > PA_MAX_SIZE || c->head_size % 8) return fail(L2B_ERR_BAD_ARG, "head_size must be a multiple of 8, at most 128");
    if (!aligned(c->dev_k) || !aligned(c->dev_v)) return fail(L2B_ERR_BAD_ARG, "pages must lie on a 16-byte boundary");
    pool.k = c->dev_k;
    pool.v = c->dev_v;
    pool.n_pages = c->n_pages;
    pool.n_kv = c->n_kv_heads;
    pool.hs = c->head_size;
    pool.page_shift = 0;
    while ((1 << pool.page_shift) < c->page_size) ++pool.page_shift;
    return L2B_OK;
}

int32_t check_batch(const l2b_paged_batch* b, const PagedPool& pool, PagedSeqs& s) {
    if (!b) return fail(L2B_ERR_BAD_ARG, "null argument");
    if (b->n_seq < 0 || b->n_query < 1 || b->pages_per_seq < 0 || b->prefix_len < 0) return fail(L2B_ERR_BAD_ARG, "bad batch shape");
    if ((b->n_seq > 0 && !b->dev_lengths) || (b->n_seq > 0 && b->pages_per_seq > 0 && !b->dev_pages) || (b->prefix_len > 0 && !b->dev_prefix_pages))
        return fail(L2B_ERR_BAD_ARG, "null argument");
    if (!aligned(b->dev_lengths, 4) || !aligned(b->dev_counts, 4) || !aligned(b->dev_pages, 4) || !aligned(b->dev_prefix_pages, 4)) return fail(L2B_ERR_BAD_ARG, "misaligned pointer");
    if (((int64_t)b->pages_per_seq << pool.page_shift) + b->prefix_len > 0x7fffffff) return fail(L2B_ERR_BAD_ARG, "more than 2^31 - 1 positions");
    if ((int64_t)b->n_seq * b->n_query > 0x7fffffff) return fail(L2B_ERR_BAD_ARG, "more than 2^31 - 1 rows");
    s.lengths = b->dev_lengths;
    s.counts = b->dev_counts;
    s.pages = b->dev_pages;
    s.prefix_pages = b->dev_prefix_pages;
    s.n_seq = b->n_seq;
    s.n_query = b->n_query;
    s.width = b->pages_per_seq;
    s.prefix_len = b->prefix_len;
    return L2B_OK;
}

int32_t check_rows(const void* p, int64_t stride, int64_t width, int type, const char* what) {
    if (!p) return fail(L2B_ERR_BAD_ARG, "null argument");
    if (stride < width) return fail(L2B_ERR_BAD_ARG, std::string(what) + ": rows overlap");
    if (!aligned(p) || stride * type_bytes(type) % 16) return fail(L2B_ERR_BAD_ARG, std::string(what) + ": rows must lie on 16-byte boundaries");
    return L2B_OK;
}

int32_t check_row_type(int type, int cache_type) {
    if (type != L2B_TYPE_F32 && type != cache_type) return fail(L2B_ERR_UNSUPPORTED_TYPE, "rows are f32 or of the cache's type");
    return L2B_OK;
}

// f(cache type, row type) with the two as types
template <typename F>
int32_t by_types(int cache_type, int type, F&& f) {
    if (cache_type == L2B_TYPE_F16) return type == L2B_TYPE_F32 ? f(__half(), float()) : f(__half(), __half());
    return type == L2B_TYPE_F32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
}

// What an attention call needs of its workspace, all in floats, and how it is cut.
struct AttnPlan {
    int blocks, smem, thin_prefix, tile_rows, slot_rows;
    PrefixCut cut;              // the prefix's own kernel, a block per SM
    int cut_blocks, stages, cut_smem;
    int64_t starts, slots, whole, cut_slots, pre, total;  // floats of the slots, of whole items, of the prefix's slots and whole items, of everything
};

// The prefix goes through the tensor cores' 128-row tiles when its rows fill more than one tile of 16; up to there it is one more group of the own
// parts' kernel, without a launch of its own.  (So it is with a negative scale, which the tiles' maxima do not allow for.)
AttnPlan attention_plan(const PagedPool& pool, const PagedSeqs& s, const l2b_paged_queries& q, int cache_type, int sms) {
    AttnPlan a;
    memset(&a, 0, sizeof(a));
    const int ks = (pool.hs + 31) / 32 * 2, n_heads = q.n_heads, group = n_heads / pool.n_kv;
    const int64_t n_tok = (int64_t)s.n_seq * s.n_query, rows = n_tok * group;
    const bool tiled = s.prefix_len > 0 && rows > 16 && q.scale >= 0.f && (int64_t)pool.n_pages * pool.n_kv < 0x7fffffff;
    a.thin_prefix = s.prefix_len > 0 && !tiled;
    const int64_t most = (int64_t)s.n_query * group * (a.thin_prefix ? s.n_seq : 1);
    a.tile_rows = most <= 8 ? 8 : 16;
    a.slot_rows = (int)(most < a.tile_rows ? most : a.tile_rows);
    const int stages = a.tile_rows == 8 ? 2 : 3;  // (ThinTraits)
    a.smem = PT_WARPS * stages * 2 * PT_KEYS * (ks * 32 + 16);
    a.blocks = sms * (a.tile_rows == 8 ? 3 : 2);
    const int64_t row = pool.hs + 4;  // sums, then maximum and total, on 16-byte boundaries
    a.slots = (int64_t)2 * a.blocks * PT_WARPS * a.slot_rows * row;
    a.whole = a.pre = s.prefix_len ? n_tok * n_heads * row : 0;
    if (tiled) {
        const bool wide = q.type == L2B_TYPE_F32;
        const int keys = wide ? 64 : 128, nd = (pool.hs + 63) / 64, terms = !wide ? 1 : cache_type == L2B_TYPE_F16 ? 2 : 3;
        a.cut.streams_share = !wide && rows > PX_ROWS ? 2 : 1;
        a.cut.tiles = (int)(((int64_t)s.prefix_len + keys - 1) / keys);
        a.cut.row_tiles = (int)((rows + PX_ROWS * a.cut.streams_share - 1) / (PX_ROWS * a.cut.streams_share));
        a.cut.units = (int64_t)a.cut.tiles * a.cut.row_tiles * pool.n_kv;
        a.cut.whole_rows = n_tok * n_heads;
        a.cut_blocks = a.cut.units < sms ? (int)a.cut.units : sms;
        a.cut.share = (a.cut.units + a.cut_blocks - 1) / a.cut_blocks;
        const int terms_bytes = terms * a.cut.streams_share * nd * PX_ROWS * 128, queries = terms_bytes > 32768 ? terms_bytes : 32768, stage = 2 * nd * keys * 128;  // (PrefixTraits)
        a.stages = (222 * 1024 - queries) / stage;  // (of 227 KB, behind barriers and a start on 1 KB)
        a.stages = a.stages < PX_MAX_STAGES ? a.stages : PX_MAX_STAGES;
        a.cut_smem = queries + a.stages * stage + 1024;
        a.cut_slots = (int64_t)2 * a.cut_blocks * 2 * PX_ROWS * row;
        a.pre *= 2 / a.cut.streams_share;
    }
    a.starts = ((int64_t)s.n_seq + a.thin_prefix + 1 + 1) / 2 * 4;  // 64-bit numbers, to a 16-byte boundary
    a.total = a.starts + a.slots + a.whole + a.cut_slots + a.pre;
    return a;
}

// Pages as rows of 64 values and as many slots as a tile takes of a page; `slots`: how many of a page's slots there are.
int32_t encode_pages(CUtensorMap* map, void* pages, const PagedPool& p, int cache_type, int keys, int slots) {
    const EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return fail(L2B_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const int page = 1 << p.page_shift;
    const cuuint64_t dims[3] = {(cuuint64_t)p.hs, (cuuint64_t)slots, (cuuint64_t)p.n_pages * p.n_kv}, strides[2] = {(cuuint64_t)p.hs * 2, (cuuint64_t)p.hs * 2 * page};
    const cuuint32_t box[3] = {64, (cuuint32_t)(page < keys ? page : keys), 1}, one[3] = {1, 1, 1};
    if (fn(map, cache_type == L2B_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, pages, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return fail(L2B_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    return L2B_OK;
}

int32_t check_queries(const l2b_paged_cache* c, const l2b_paged_queries* q, const PagedSeqs& s) {
    if (!q) return fail(L2B_ERR_BAD_ARG, "null argument");
    L2B_TRY(check_row_type(q->type, c->type));
    if (q->n_heads <= 0 || q->n_heads > 65535 || q->n_heads % c->n_kv_heads) return fail(L2B_ERR_BAD_ARG, "n_heads must be a multiple of n_kv_heads");
    if ((int64_t)s.n_seq * s.n_query * q->n_heads > 0x7fffffff) return fail(L2B_ERR_BAD_ARG, "more than 2^31 - 1 query heads");
    if (!std::isfinite(q->scale * LOG2E)) return fail(L2B_ERR_BAD_ARG, "scale must be at most 2.3e38 in size, or 0 for 1 / sqrt(head_size)");
    return L2B_OK;
}

}  // namespace

extern "C" int32_t l2b_paged_append_device(const l2b_paged_cache* cache, const l2b_paged_batch* batch, const l2b_paged_rows* rows, void* stream) {
    AppendParams p;
    memset(&p, 0, sizeof(p));
    L2B_TRY(check_cache(cache, p.pool));
    L2B_TRY(check_batch(batch, p.pool, p.seqs));
    if (!rows) return fail(L2B_ERR_BAD_ARG, "null argument");
    L2B_TRY(check_row_type(rows->type, cache->type));
    const int hs = p.pool.hs;
    if ((rows->dev_q == nullptr) != (rows->dev_q_out == nullptr)) return fail(L2B_ERR_BAD_ARG, "dev_q and dev_q_out go together");
    if (rows->dev_q) {
        if (rows->n_heads <= 0 || rows->n_heads > 65535) return fail(L2B_ERR_BAD_ARG, "bad number of heads");
        L2B_TRY(check_rows(rows->dev_q, rows->q_stride, (int64_t)rows->n_heads * hs, rows->type, "dev_q"));
        L2B_TRY(check_rows(rows->dev_q_out, rows->q_out_stride, (int64_t)rows->n_heads * hs, rows->type, "dev_q_out"));
        if (rows->dev_q == rows->dev_q_out && rows->q_stride != rows->q_out_stride) return fail(L2B_ERR_BAD_ARG, "in place the strides must be the same");
    }
    L2B_TRY(check_rows(rows->dev_k, rows->k_stride, (int64_t)p.pool.n_kv * hs, rows->type, "dev_k"));
    L2B_TRY(check_rows(rows->dev_v, rows->v_stride, (int64_t)p.pool.n_kv * hs, rows->type, "dev_v"));
    if (!aligned(rows->dev_q_gain) || !aligned(rows->dev_k_gain)) return fail(L2B_ERR_BAD_ARG, "gains must lie on a 16-byte boundary");
    if ((rows->dev_q_gain || rows->dev_k_gain) && !(rows->eps >= 0.f)) return fail(L2B_ERR_BAD_ARG, "eps must not be negative");
    if (!(rows->rope_freq_base >= 0.f) || std::isinf(rows->rope_freq_base)) return fail(L2B_ERR_BAD_ARG, "rope_freq_base must be positive, or 0 for no rotation");
    p.q = rows->dev_q; p.k = rows->dev_k; p.v = rows->dev_v; p.q_out = rows->dev_q_out;
    p.q_stride = rows->q_stride; p.k_stride = rows->k_stride; p.v_stride = rows->v_stride; p.q_out_stride = rows->q_out_stride;
    p.q_gain = rows->dev_q_gain; p.k_gain = rows->dev_k_gain; p.eps = rows->eps; p.inv_size = 1.f / (float)hs;
    p.n_heads = rows->n_heads;
    const bool rotate = rows->rope_freq_base > 0.f;
    if (rotate) {
        const long double step = powl((long double)rows->rope_freq_base, -2.0L / hs);
        long double f = 0.15915494309189533576888376337251436L;  // turns per radian
        for (int i = 0; i < hs / 2; ++i, f *= step) p.turns[i] = (double)f;
    }
    OnDeviceOf on;
    L2B_TRY(on.enter(cache->dev_k, "dev_k"));
    const int64_t n = (int64_t)p.seqs.n_seq * p.seqs.n_query;
    if (n == 0) return L2B_OK;
    // Tokens of a block: their angles are worked out together, so as many tokens as the block has warps once there are blocks enough for every SM three
    // times over; before that fewer, and their heads over several warps, at last over several blocks.
    int sms = 0;
    L2B_TRY(sm_count(on.device, &sms));
    p.tokens = PA_WARPS;
    while (p.tokens > 1 && n < (int64_t)3 * sms * p.tokens) p.tokens /= 2;
    const int piece = hs % 16 ? 4 : 8;
    int lanes = 1;
    while (lanes < hs / (2 * piece)) lanes *= 2;
    const int at_once = 32 / lanes, groups = ((p.q ? p.n_heads : 0) + at_once - 1) / at_once + 2 * ((p.pool.n_kv + at_once - 1) / at_once);
    const int64_t blocks = (n + p.tokens - 1) / p.tokens;
    int y = 1;
    while (y * (PA_WARPS / p.tokens) < groups && y < 64 && blocks * y < 2 * sms) ++y;
    const dim3 grid((unsigned)blocks, (unsigned)y);
    return by_types(cache->type, rows->type, [&](auto t, auto io) -> int32_t {
        using T = decltype(t);
        using TIO = decltype(io);
        cudaStream_t st = (cudaStream_t)stream;
        auto go = [&](auto kernel) -> int32_t {
            CU(launch_kernel(kernel, grid, dim3(PA_THREADS), 0, st, true, p));
            return L2B_OK;
        };
        auto pairs = [&](auto size) -> int32_t {
            constexpr int P = decltype(size)::value;
            if (!rotate) return go(paged_append_kernel<TIO, T, P, PAIRS_NONE>);
            return rows->rope_is_neox ? go(paged_append_kernel<TIO, T, P, PAIRS_HALF_APART>) : go(paged_append_kernel<TIO, T, P, PAIRS_NEIGHBOURS>);
        };
        L2B_TRY(piece == 8 ? pairs(std::integral_constant<int, 8>()) : pairs(std::integral_constant<int, 4>()));
        return L2B_OK;
    });
}

extern "C" int32_t l2b_paged_attention_workspace(const l2b_paged_cache* cache, const l2b_paged_batch* batch, const l2b_paged_queries* queries, int64_t* bytes) {
    PagedPool pool;
    PagedSeqs seqs;
    L2B_TRY(check_cache(cache, pool));
    L2B_TRY(check_batch(batch, pool, seqs));
    L2B_TRY(check_queries(cache, queries, seqs));
    if (!bytes) return fail(L2B_ERR_BAD_ARG, "null argument");
    OnDeviceOf on;
    L2B_TRY(on.enter(cache->dev_k, "dev_k"));
    int sms = 0;
    L2B_TRY(sm_count(on.device, &sms));
    *bytes = attention_plan(pool, seqs, *queries, cache->type, sms).total * 4;
    return L2B_OK;
}

extern "C" int32_t l2b_paged_attention_device(const l2b_paged_cache* cache, const l2b_paged_batch* batch, const l2b_paged_queries* queries, void* dev_workspace,
                                              int64_t workspace_bytes, void* stream) {
    PagedAttnParams p;
    memset(&p, 0, sizeof(p));
    L2B_TRY(check_cache(cache, p.pool));
    L2B_TRY(check_batch(batch, p.pool, p.seqs));
    L2B_TRY(check_queries(cache, queries, p.seqs));
    const int hs = p.pool.hs;
    L2B_TRY(check_rows(queries->dev_q, queries->q_stride, (int64_t)queries->n_heads * hs, queries->type, "dev_q"));
    L2B_TRY(check_rows(queries->dev_out, queries->out_stride, (int64_t)queries->n_heads * hs, queries->type, "dev_out"));
    OnDeviceOf on;
    L2B_TRY(on.enter(cache->dev_k, "dev_k"));
    if (p.seqs.n_seq == 0) return L2B_OK;
    int sms = 0;
    L2B_TRY(sm_count(on.device, &sms));
    const AttnPlan plan = attention_plan(p.pool, p.seqs, *queries, cache->type, sms);
    if (!dev_workspace || !aligned(dev_workspace) || workspace_bytes < plan.total * 4)
        return fail(L2B_ERR_BAD_ARG, "the workspace must lie on a 16-byte boundary and hold l2b_paged_attention_workspace bytes");
    p.q = queries->dev_q; p.out = queries->dev_out; p.q_stride = queries->q_stride; p.out_stride = queries->out_stride;
    p.n_heads = queries->n_heads;
    p.group = queries->n_heads / p.pool.n_kv;
    p.scale2 = (queries->scale != 0.f ? queries->scale : 1.f / sqrtf((float)hs)) * LOG2E;
    p.thin_prefix = plan.thin_prefix;
    p.cut = plan.cut;
    p.workers = plan.blocks * PT_WARPS;
    p.slot_rows = plan.slot_rows;
    p.tile_shift = plan.tile_rows == 8 ? 3 : 4;
    p.starts = (int64_t*)dev_workspace;
    float* const w = (float*)dev_workspace + plan.starts;
    const int64_t n_rows = (int64_t)p.seqs.n_seq * p.seqs.n_query * p.n_heads;
    p.slot_acc = w;
    p.slot_ml = w + (int64_t)2 * p.workers * p.slot_rows * hs;
    if (p.seqs.prefix_len) {
        p.own_acc = w + plan.slots;
        p.own_ml = p.own_acc + n_rows * hs;
        p.cut_acc = p.own_acc + plan.whole;
        p.cut_ml = p.cut_acc + (int64_t)2 * plan.cut_blocks * 2 * PX_ROWS * hs;
        p.pre_acc = p.cut_acc + plan.cut_slots;
        p.pre_ml = p.pre_acc + n_rows * hs * (plan.cut.streams_share == 1 ? 2 : 1);
    }
    cudaStream_t st = (cudaStream_t)stream;
    L2B_TRY(by_types(cache->type, queries->type, [&](auto t, auto io) -> int32_t {
        using T = decltype(t);
        using TIO = decltype(io);
        if (plan.cut.units > 0) {
            PrefixParams x;
            memset(&x, 0, sizeof(x));
            static_cast<PagedWork&>(x) = p;
            x.q = p.q; x.q_stride = p.q_stride; x.n_heads = p.n_heads;
            x.rows = p.seqs.n_seq * p.seqs.n_query * p.group;
            x.stages = plan.stages;
            x.scale2 = p.scale2;
            x.cut = plan.cut;
            x.slot_acc = p.cut_acc; x.slot_ml = p.cut_ml; x.pre_acc = p.pre_acc; x.pre_ml = p.pre_ml;
            const int keys = sizeof(TIO) == 4 ? 64 : 128, page = 1 << p.pool.page_shift;
            CUtensorMap mk, mv, me;
            L2B_TRY(encode_pages(&mk, p.pool.k, p.pool, cache->type, keys, page));
            L2B_TRY(encode_pages(&mv, p.pool.v, p.pool, cache->type, keys, page));
            L2B_TRY(encode_pages(&me, p.pool.v, p.pool, cache->type, keys, (p.seqs.prefix_len - 1) % page + 1));
            auto tiled = [&](auto tiles) -> int32_t {
                constexpr int TILES = decltype(tiles)::value;
                L2B_TRY((allow_smem<paged_prefix_kernel<T, TIO, TILES>>(on.device)));
                CU(launch_kernel_args(paged_prefix_kernel<T, TIO, TILES>, dim3((unsigned)plan.cut_blocks), dim3(PX_THREADS), (size_t)plan.cut_smem, st, true, 1, x, mk, mv, me));
                return L2B_OK;
            };
            if constexpr (sizeof(TIO) == 4) {
                L2B_TRY(tiled(std::integral_constant<int, 1>()));
            } else if (plan.cut.streams_share == 2) {
                L2B_TRY(tiled(std::integral_constant<int, 2>()));
            } else {
                L2B_TRY(tiled(std::integral_constant<int, 1>()));
            }
        }
        auto go = [&](auto ks, auto nt) -> int32_t {
            constexpr int KS = decltype(ks)::value, NT = decltype(nt)::value;
            L2B_TRY((allow_smem<paged_attention_kernel<T, TIO, KS, NT>>(on.device)));
            CU(launch_kernel(paged_attention_kernel<T, TIO, KS, NT>, dim3((unsigned)plan.blocks), dim3(PT_WARPS * 32), (size_t)plan.smem, st, true, p));
            return L2B_OK;
        };
        auto size = [&](auto nt) -> int32_t {
            switch ((hs + 31) / 32) {
                case 1: return go(std::integral_constant<int, 2>(), nt);
                case 2: return go(std::integral_constant<int, 4>(), nt);
                case 3: return go(std::integral_constant<int, 6>(), nt);
                default: return go(std::integral_constant<int, 8>(), nt);
            }
        };
        L2B_TRY(plan.tile_rows == 8 ? size(std::integral_constant<int, 1>()) : size(std::integral_constant<int, 2>()));
        JoinParams j;
        j.a = p;
        // A warp per row once there are rows for a few warps on every SM, else the block's eight share one.  Whole calls, eight warps / one, 32 heads of 128 values: own
        // positions alone (1 500 each) 256 rows 16.8 / 22.8 us, 768 31.5 / 31.3, 1 024 37.5 / 36.0, 2 048 59.4 / 51.4; behind a prefix of 6 001, whose parts are
        // more, 256 rows 33 / 40, 768 42 / 48, 1 024 47 / 51, 1 536 55 / 54, 2 048 64 / 60.  The border lies between the two kinds'.
        j.heads = n_rows >= 1024 ? PJ_WARPS : 1;
        const dim3 grid((unsigned)(p.seqs.n_seq * p.seqs.n_query), (unsigned)((p.n_heads + j.heads - 1) / j.heads));
        CU(launch_kernel(paged_join_kernel<TIO>, grid, dim3(PJ_WARPS * 32), 0, st, true, j));
        return L2B_OK;
    }));
    return L2B_OK;
}

// Blocks of a row: as many as keep a slice at 16384 logits (two blocks to an SM), more while SMs would be idle and a slice has work for the block.
template <typename T>
static int32_t launch_sample(SampleParams& p, int n_rows, int device, cudaStream_t st) {
    int sms = 0;
    L2B_TRY(sm_count(device, &sms));
    int cluster = 1;
    while (cluster < FS_CLUSTER && ((p.vocab + cluster - 1) / cluster > 16384 || ((int64_t)n_rows * cluster * 2 <= 2 * sms && p.vocab / cluster >= 4096))) cluster *= 2;
    p.cluster = cluster;
    p.slice = ((p.vocab + cluster - 1) / cluster + 7) / 8 * 8;
    L2B_TRY(allow_smem<filtered_sample_kernel<T>>(device));
    CU(launch_kernel(filtered_sample_kernel<T>, dim3((unsigned)(n_rows * cluster)), dim3(FS_THREADS), (size_t)p.slice * 4, st, true, p, cluster));
    return L2B_OK;
}

extern "C" int32_t l2b_sample_device(const l2b_sampling* a, void* stream) {
    if (!a || !a->dev_logits || !a->dev_tokens || !a->dev_uniform) return fail(L2B_ERR_BAD_ARG, "null argument");
    if (a->type != L2B_TYPE_F32 && a->type != L2B_TYPE_F16 && a->type != L2B_TYPE_BF16) return fail(L2B_ERR_UNSUPPORTED_TYPE, "logits are f32, f16 or bf16");
    if (a->n_rows < 0 || a->vocab < 1 || a->vocab > SAMPLE_MAX_VOCAB) return fail(L2B_ERR_BAD_ARG, "bad number of rows, or a vocabulary of more than 393216");
    if (a->n_rows > 0x7fffffff / FS_CLUSTER) return fail(L2B_ERR_BAD_ARG, "too many rows");
    if (a->stride < a->vocab) return fail(L2B_ERR_BAD_ARG, "rows overlap");
    if (!aligned(a->dev_logits, type_bytes(a->type)) || !aligned(a->dev_tokens, 4) || !aligned(a->dev_uniform, 8) || !aligned(a->dev_temperature, 4) || !aligned(a->dev_top_k, 4) ||
        !aligned(a->dev_top_p, 4) || !aligned(a->dev_min_p, 4) || !aligned(a->dev_probs, 4))
        return fail(L2B_ERR_BAD_ARG, "misaligned pointer");
    OnDeviceOf on;
    L2B_TRY(on.enter(a->dev_logits, "dev_logits"));
    if (a->n_rows == 0) return L2B_OK;
    SampleParams p;
    memset(&p, 0, sizeof(p));
    p.logits = a->dev_logits; p.stride = a->stride; p.vocab = a->vocab;
    p.temperature = a->dev_temperature; p.top_p = a->dev_top_p; p.min_p = a->dev_min_p; p.top_k = a->dev_top_k;
    p.same_temperature = p.same_top_p = 1.f;
    p.uniform = a->dev_uniform; p.tokens = a->dev_tokens; p.probs = a->dev_probs;
    cudaStream_t st = (cudaStream_t)stream;
    return a->type == L2B_TYPE_F32 ? launch_sample<float>(p, a->n_rows, on.device, st)
                                   : a->type == L2B_TYPE_F16 ? launch_sample<__half>(p, a->n_rows, on.device, st) : launch_sample<__nv_bfloat16>(p, a->n_rows, on.device, st);
}

int32_t enqueue_filtered_sample(const float* logits, int vocab, float temperature, int top_k, float top_p, float min_p, double uniform, int* token, int device, cudaStream_t st) {
    SampleParams p;
    memset(&p, 0, sizeof(p));
    p.logits = logits; p.stride = vocab; p.vocab = vocab; p.tokens = token;
    p.same_temperature = temperature; p.same_top_k = top_k; p.same_top_p = top_p; p.same_min_p = min_p; p.same_uniform = uniform;
    return launch_sample<float>(p, 1, device, st);
}
