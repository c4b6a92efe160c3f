// mars_attn.cu -- attention of each request's new tokens over its cache pages.
// First form: one warp for each (token, query head), one key at a time.
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <string>

#include "mars_attn.cuh"
#include "mars_attn_mma.cuh"
#include "mars_kv.h"

using namespace mars;

namespace {

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__global__ void __launch_bounds__(128) attn_rows_kernel(const AttnArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= (int64_t)a.T * a.hq) return;
    const int t = (int)(w / a.hq), h = (int)(w % a.hq);
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu_new[mid] <= t) lo = mid; else hi = mid;
    }
    const Request r = load_request(a, lo);
    if (t < r.first || t >= r.first + r.rows) return;
    int low, high;
    row_range(a, r, t - r.first, t - r.first + 1, &low, &high);
    const int pos = r.len - r.rows + (t - r.first);
    const T* q = reinterpret_cast<const T*>(a.q) + t * a.q_tok + h * a.q_head;
    float qv[4], acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        acc[i] = 0.0f;
        qv[i] = lane + 32 * i < a.D ? to_f(q[lane + 32 * i]) : 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    const float decay = a.decay != nullptr ? a.decay[h] : 0.0f;
    for (int j = 0; j < high; ++j) {
        if (j >= r.prefix && j < low) { j = low - 1; continue; }
        const int page = a.tables[(int64_t)lo * a.pitch + j / a.page];
        const bool there = page >= 0 && page < a.num_pages;
        const T* k = reinterpret_cast<const T*>(a.k) + page * a.k_page + (j % a.page) * a.k_slot + (h / a.group) * a.k_head;
        const T* v = reinterpret_cast<const T*>(a.v) + page * a.v_page + (j % a.page) * a.v_slot + (h / a.group) * a.v_head;
        float s = 0.0f, vv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = there && lane + 32 * i < a.D;
            vv[i] = in ? to_f(v[lane + 32 * i]) : 0.0f;
            s += in ? qv[i] * to_f(k[lane + 32 * i]) : 0.0f;
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        s *= a.scale;
        if (a.cap > 0.0f) s = a.cap * tanh_exp(s / a.cap);
        s -= decay * (float)max(0, pos - j);
        const float mm = fmaxf(m, s), keep = __expf(m - mm), p = __expf(s - mm);
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = acc[i] * keep + p * vv[i];
        m = mm;
    }
    T* o = reinterpret_cast<T*>(a.out) + t * a.o_tok + h * a.o_head;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < a.D) o[lane + 32 * i] = from_f<T>(l > 0.0f ? acc[i] / l : 0.0f);
    if (lane == 0 && a.lse != nullptr) a.lse[w] = l > 0.0f ? m + logf(l) : -INFINITY;
}

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
    const struct { CUtensorMap* map; void* base; int64_t slot, head, page; } side[2] = {
        {k, c->k, c->k_slot_stride, c->k_head_stride, c->k_page_stride},
        {v, c->v, c->v_slot_stride, c->v_head_stride, c->v_page_stride}};
    for (const auto& s : side) {
        const cuuint64_t stride[3] = {(cuuint64_t)s.slot * 2, (cuuint64_t)s.head * 2, (cuuint64_t)s.page * 2};
        const CUresult r = enc(s.map, type, 4, s.base, dim, stride, shape, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS)
            return fail(MARS_ERR_INVALID, "mars_paged_attention: the cache's strides make no tensor map (" +
                                              std::to_string((int)r) + ")");
    }
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
    if (q_heads / cache->kv_heads > MARS_ATTN_MAX_GROUP)
        return fail(MARS_ERR_UNSUPPORTED, fn + ": at most " + std::to_string(MARS_ATTN_MAX_GROUP) + " query heads a key head");
    if (!std::isfinite(cfg->scale) || !(cfg->softcap >= 0.0f) || !std::isfinite(cfg->softcap) || cfg->window < 0)
        return fail(MARS_ERR_INVALID, fn + ": scale must be finite, softcap and window finite and not negative");
    if (tokens == 0 || B == 0) return MARS_OK;
    if (d_q == nullptr || d_cu_new == nullptr || d_kv_lens == nullptr || d_tables == nullptr || d_out == nullptr)
        return fail(MARS_ERR_INVALID, fn + ": NULL argument");
    const uintptr_t bases = reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_out) |
                            reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v);
    const int64_t strides = q_token_stride | q_head_stride | out_token_stride | out_head_stride | cache->k_page_stride |
                            cache->k_slot_stride | cache->k_head_stride | cache->v_page_stride | cache->v_slot_stride |
                            cache->v_head_stride;
    if ((bases & 15) != 0 || strides % 8 != 0)
        return fail(MARS_ERR_INVALID, fn + ": q, out, k and v must start on 16 bytes and have strides of multiples of 16 bytes");
    MarsDeviceGuard g(c->device);
    cudaStream_t st;
    MARS_TRY(kv_begin(c, stream, &st));
    AttnArgs a{};
    a.q = d_q; a.out = d_out; a.lse = d_lse; a.k = cache->k; a.v = cache->v;
    a.cu_new = d_cu_new; a.kv_lens = d_kv_lens; a.tables = d_tables; a.prefix = d_prefix_lens; a.decay = d_decay;
    a.q_tok = q_token_stride; a.q_head = q_head_stride; a.o_tok = out_token_stride; a.o_head = out_head_stride;
    a.k_page = cache->k_page_stride; a.k_slot = cache->k_slot_stride; a.k_head = cache->k_head_stride;
    a.v_page = cache->v_page_stride; a.v_slot = cache->v_slot_stride; a.v_head = cache->v_head_stride;
    a.scale = cfg->scale; a.cap = cfg->softcap; a.window = cfg->window;
    a.T = tokens; a.B = B; a.hq = q_heads; a.hkv = cache->kv_heads; a.group = q_heads / cache->kv_heads;
    a.D = cache->head_dim; a.page = cache->page_size; a.num_pages = cache->num_pages; a.pitch = table_pitch;
    AttnWork w{};
    w.part_o = c->d_part_o; w.part_ml = c->d_part_ml; w.tickets = c->d_tickets + kKvTickets; w.err = c->d_err;
    w.host_err = c->h_err;
    if ((int64_t)std::max(cfg->max_new, 1) * a.group <= kShortRows) {
        MARS_TRY(attn_short(a, w, cache, c->num_sms, st));
        return kv_end(c, st);
    }
    const unsigned grid = (unsigned)(((int64_t)tokens * q_heads + 3) / 4);
    if (cache->dtype == MARS_DTYPE_F16) attn_rows_kernel<__half><<<grid, 128, 0, st>>>(a);
    else attn_rows_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a);
    MARS_CUDA_TRY(cudaGetLastError());
    return kv_end(c, st);
}
