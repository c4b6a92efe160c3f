// mars_attn.cu -- attention of each request's new tokens over its cache pages:
// the entry point, its checks, the choice of the kernel and the tensor maps.
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <string>

#include "mars_attn.cuh"
#include "mars_attn_mma.cuh"
#include "mars_kv.h"

using namespace mars;

namespace {

PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

Cap make_cap(float scale, float softcap) {
    constexpr float kMost = 3.402823466e38f, kLog2e = 1.4426950408889634f;
    const float fit[6] = {1.0f, -0.333333283662796f, 0.13332964479923248f, -0.053899191319942474f, 0.021297989413142204f,
                          -0.006647486239671707f};
    Cap t{};
    if (softcap == 0.0f) return t;
    t.in = std::min(std::max(scale / softcap, -kMost), kMost);      // finite: 0 times it is 0
    t.out = std::min(softcap * kLog2e, kMost);
    float power = scale * kLog2e, c = 0.0f;                // in * out, also where those are at the type's ends
    for (int k = 0; k < 6; ++k) {
        c = fit[k] * power;
        uint32_t bits;
        memcpy(&bits, &c, 4);
        t.c[k] = (uint64_t)bits << 32 | bits;
        power *= t.in * t.in;
    }
    // s * s is finite up to 1e18.  A cap so small that the powers overflow: its scores are
    // next to nothing, tanh_exp's error with them.
    t.most = std::isfinite(c) ? std::min(0.5f / std::fabs(t.in), 1e18f) : -1.0f;
    return t;
}

}  // namespace

namespace mars {

int page_box(int page, int tile) {
    int box = 8;                              // page sizes are multiples of 8
    while (box * 2 <= tile && page % (box * 2) == 0) box *= 2;
    return box;
}

// dimensions: column, token of the page, head, page; out of range reads as 0
int page_maps(const mars_kv_cache* c, int box, CUtensorMap* k, CUtensorMap* v) {
    auto enc = get_encode();
    if (enc == nullptr) return fail(MARS_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dim[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size, (cuuint64_t)c->kv_heads,
                               (cuuint64_t)c->num_pages};
    const cuuint32_t shape[4] = {64, (cuuint32_t)box, 1, 1}, unit[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type =
        c->dtype == MARS_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    // A key is one piece of memory; where it is 128 bytes, fetching 256 would read its
    // neighbour head's too, which another CTA wants at another time (64 requests of up
    // to 16,000 keys, 8 key heads of 64 columns: 229 us with 128, 299 with 256).
    const CUtensorMapL2promotion fetch =
        c->head_dim <= 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
    const struct { CUtensorMap* map; void* base; int64_t slot, head, page; } side[2] = {
        {k, c->k, c->k_slot_stride, c->k_head_stride, c->k_page_stride},
        {v, c->v, c->v_slot_stride, c->v_head_stride, c->v_page_stride}};
    for (const auto& s : side) {
        const cuuint64_t stride[3] = {(cuuint64_t)s.slot * 2, (cuuint64_t)s.head * 2, (cuuint64_t)s.page * 2};
        const CUresult r = enc(s.map, type, 4, s.base, dim, stride, shape, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, fetch,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS)
            return fail(MARS_ERR_INVALID, "mars_paged_attention: the cache's strides make no tensor map (" +
                                              std::to_string((int)r) + ")");
    }
    return MARS_OK;
}

// dimensions: column, query head of a key head, key head, token
int query_map(const AttnArgs& a, int32_t dtype, int tokens, CUtensorMap* q) {
    auto enc = get_encode();
    if (enc == nullptr) return fail(MARS_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dim[4] = {(cuuint64_t)a.D, (cuuint64_t)a.group, (cuuint64_t)a.hkv, (cuuint64_t)a.T};
    const cuuint64_t stride[3] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_head * a.group * 2, (cuuint64_t)a.q_tok * 2};
    const cuuint32_t shape[4] = {64, (cuuint32_t)a.group, 1, (cuuint32_t)tokens}, unit[4] = {1, 1, 1, 1};
    const CUresult r = enc(q, dtype == MARS_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                           4, const_cast<void*>(a.q), dim, stride, shape, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(MARS_ERR_INVALID, "mars_paged_attention: q's strides make no tensor map (" + std::to_string((int)r) + ")");
    return MARS_OK;
}

int allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    MARS_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if ((done.load(std::memory_order_relaxed) & bit) != 0) return MARS_OK;
    MARS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit);
    return MARS_OK;
}

}  // namespace mars

extern "C" int mars_paged_attention(mars_kv_ctx* c, const mars_kv_cache* cache, const void* d_q,
                                    int64_t q_token_stride, int64_t q_head_stride, int32_t tokens, int32_t q_heads,
                                    int32_t B, const int32_t* d_cu_new, const int32_t* d_kv_lens,
                                    const int32_t* d_tables, int32_t table_pitch, const mars_attn_config* cfg,
                                    const float* d_decay, const int32_t* d_prefix_lens, void* d_out,
                                    int64_t out_token_stride, int64_t out_head_stride, float* d_lse, void* stream) {
    const std::string fn = "mars_paged_attention";
    if (c == nullptr || cfg == nullptr) return fail(MARS_ERR_INVALID, fn + ": NULL context or configuration");
    MARS_TRY(check_cache(cache, fn.c_str()));
    if (B < 0 || B > c->max_requests)
        return fail(MARS_ERR_CAPACITY, fn + ": B must be in [0, " + std::to_string(c->max_requests) + "]");
    if (tokens < 0 || table_pitch <= 0 || q_heads <= 0 || q_heads % cache->kv_heads != 0)
        return fail(MARS_ERR_INVALID, fn + ": tokens must not be negative, table_pitch positive, q_heads a multiple of kv_heads");
    if (cache->head_dim % 8 != 0 || cache->head_dim > MARS_ATTN_MAX_HEAD_DIM || cache->page_size % 8 != 0)
        return fail(MARS_ERR_UNSUPPORTED, fn + ": head_dim must be a multiple of 8 up to " +
                                              std::to_string(MARS_ATTN_MAX_HEAD_DIM) + ", page_size a multiple of 8");
    if ((int64_t)cache->num_pages * cache->page_size > MARS_ATTN_MAX_KEYS)
        return fail(MARS_ERR_UNSUPPORTED, fn + ": at most " + std::to_string(MARS_ATTN_MAX_KEYS) + " tokens a cache");
    if (q_heads / cache->kv_heads > MARS_ATTN_MAX_GROUP)
        return fail(MARS_ERR_UNSUPPORTED, fn + ": at most " + std::to_string(MARS_ATTN_MAX_GROUP) + " query heads a key head");
    if (!std::isfinite(cfg->scale) || !(cfg->softcap >= 0.0f) || !std::isfinite(cfg->softcap) || cfg->window < 0)
        return fail(MARS_ERR_INVALID, fn + ": scale must be finite, softcap and window finite and not negative");
    if (tokens == 0 || B == 0) return MARS_OK;
    if (d_q == nullptr || d_cu_new == nullptr || d_kv_lens == nullptr || d_tables == nullptr || d_out == nullptr)
        return fail(MARS_ERR_INVALID, fn + ": NULL argument");
    // the stride of a dimension of one entry says nothing
    mars_kv_cache kv = *cache;
    if (q_heads == 1) q_head_stride = out_head_stride = kv.head_dim;
    if (tokens == 1) q_token_stride = out_token_stride = (int64_t)q_heads * kv.head_dim;
    if (kv.kv_heads == 1) kv.k_head_stride = kv.v_head_stride = kv.head_dim;
    if (kv.num_pages == 1) kv.k_page_stride = kv.v_page_stride = kv.head_dim;
    cache = &kv;
    const uintptr_t bases = reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_out) |
                            reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v);
    const int64_t strides = q_token_stride | q_head_stride | out_token_stride | out_head_stride | cache->k_page_stride |
                            cache->k_slot_stride | cache->k_head_stride | cache->v_page_stride | cache->v_slot_stride |
                            cache->v_head_stride;
    if ((bases & 15) != 0 || strides % 8 != 0 || strides < 0)
        return fail(MARS_ERR_INVALID,
                    fn + ": q, out, k and v must start on 16 bytes and have strides of multiples of 16 bytes, not negative");
    MarsDeviceGuard g(c->device);
    cudaStream_t st;
    MARS_TRY(kv_begin(c, stream, &st));
    AttnArgs a{};
    a.q = d_q; a.out = d_out; a.lse = d_lse;
    a.cu_new = d_cu_new; a.kv_lens = d_kv_lens; a.tables = d_tables; a.prefix = d_prefix_lens; a.decay = d_decay;
    a.q_tok = q_token_stride; a.q_head = q_head_stride; a.o_tok = out_token_stride; a.o_head = out_head_stride;
    a.scale = cfg->scale; a.softcap = cfg->softcap; a.cap = make_cap(cfg->scale, cfg->softcap); a.window = cfg->window;
    a.T = tokens; a.B = B; a.hq = q_heads; a.hkv = cache->kv_heads; a.group = q_heads / cache->kv_heads;
    a.D = cache->head_dim; a.page = cache->page_size; a.num_pages = cache->num_pages; a.pitch = table_pitch;
    // The short kernel's tiles have 16 rows: with more it would read the keys once for
    // every 16, the chunk kernel once for every 256 but with three launches and tiles
    // of 128 rows (64 ragged requests, 4 query heads a key head: 4 new tokens 208 us
    // here, 5 there 273; 4 requests of 700 keys on the device: 11 us and 18).
    const bool chunk = (int64_t)std::max(cfg->max_new, 1) * a.group > kShortRows;
    MARS_TRY(kv_attn_memory(c, chunk));
    AttnWork w{};
    w.part_o = c->d_part_o; w.part_ml = c->d_part_ml; w.tickets = c->d_tickets + kKvTickets;
    w.host_err = c->h_err; w.chunk_o = c->d_chunk_o; w.chunk_ml = c->d_chunk_ml; w.starts = c->d_starts;
    w.failed = c->d_failed;
    w.wait_ns = c->wait_ns; w.stall = c->stall ? 0 : -1;
    c->stall = false;
    const int done = chunk ? attn_chunk(a, w, cache, c->num_sms, st) : attn_short(a, w, cache, c->num_sms, st);
    const int end = kv_end(c, st);                 // also after an error: some launches may be under way
    return done != MARS_OK ? done : end;
}
