// mars_rope.cu -- rotary positions with several axes (time, height, width of
// an image or a video; one axis for text), alone in both directions and fused
// with the write of keys and values into their cache pages.
//
// Pair i of a head is turned by angle = position[token][axis[i]] * freq[i]:
//     (a, b) -> (a cos - b sin, a sin + b cos),
// where (a, b) are columns (i, i + rot/2), or (2i, 2i + 1) when interleaved;
// columns from rot on are copied.  The rotation R is orthogonal, so the
// gradient of y = R x is R^T dy: the same kernel with the angle negated.
//
// The angle is formed in 64 bits and reduced to [-1, 1] turns of pi before it
// is rounded, because position * freq rounded to 32 bits loses 2^-24 of the
// whole angle: 0.002 rad at position 32,768.  A token's angles are computed
// once for all its heads (shared memory), a few 64-bit operations for each of
// the rot/2 pairs.
//
// Bound: HBM (every value is read and written once).  A block takes 1 to 4
// tokens; threadIdx.x walks the 16-byte chunks of a head, threadIdx.y the
// heads of q, k and v of all the block's tokens, so a warp covers whole
// 128-byte lines on both sides; each thread has two 16-byte loads in flight,
// and 1,536 threads an SM (of 2,048: 33 to 40 registers) cover the latency.
// Measured: 8,192 tokens of 32 + 8 + 8 heads of 128 in bf16 41 us, 4.9 TB/s, 0.76
// of the copy rate; 16,381 tokens of 12 heads of 64 in fp32 20.6 us, 0.76.  Halves
// that no 16-byte vector divides (72 or 120 columns in 16 bits) go by single
// elements: the same 8,192 tokens with heads of 120 95 us, 0.31, of 72 83 us, 0.21.  Loads issued one item ahead of the
// stores, the first beside the angles, were slower (53 us: more registers,
// fewer blocks).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "mars_kv.h"

using namespace mars;

namespace {

constexpr int kThreads = 256;              // of a block at most
constexpr int kMaxTokens = 4;          // tokens of one block
constexpr int kMaxHalf = 512;          // pairs of a head

struct Rows {
    const char* src;                   // bytes; token and head strides in elements
    char* dst;
    int64_t src_tok, src_head, dst_tok, dst_head;
};

struct RopeArgs {
    Rows q, k, v;                      // k.dst / v.dst: the cache; dst_tok unused there
    int64_t k_page, k_slot, v_page, v_slot;
    const int32_t* slots;              // NULL: no cache (q only)
    const int32_t* positions;
    const float* freq;
    const int32_t* axis;
    int64_t slots_in_cache;
    int32_t T, hq, hkv, D, half, axes, page, tokens_per_block;
    float sign;                        // -1: the inverse rotation
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

template <typename T, int V> struct alignas(sizeof(T) * V) Chunk { T e[V]; };

// Turns the pairs (a.e[i], b.e[i]) by (cos, sin) = cs[i].
template <typename T, int V>
__device__ __forceinline__ void turn_split(Chunk<T, V>& a, Chunk<T, V>& b, const float2* cs) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float x = to_f(a.e[i]), y = to_f(b.e[i]);
        a.e[i] = from_f<T>(x * cs[i].x - y * cs[i].y);
        b.e[i] = from_f<T>(x * cs[i].y + y * cs[i].x);
    }
}

// Turns the neighbouring pairs inside a chunk.
template <typename T, int V>
__device__ __forceinline__ void turn_inside(Chunk<T, V>& a, const float2* cs) {
#pragma unroll
    for (int i = 0; i + 1 < V; i += 2) {
        const float x = to_f(a.e[i]), y = to_f(a.e[i + 1]);
        a.e[i] = from_f<T>(x * cs[i / 2].x - y * cs[i / 2].y);
        a.e[i + 1] = from_f<T>(x * cs[i / 2].y + y * cs[i / 2].x);
    }
}

// One head: item p of it, two chunks.  half = 0: a plain copy.
template <typename T, int V, bool kInterleaved>
__device__ __forceinline__ void head_items(const T* src, T* dst, int D, int half,
                                           const float2* cs, int x0, int xstep) {
    using C = Chunk<T, V>;
    const C* s = reinterpret_cast<const C*>(src);
    C* d = reinterpret_cast<C*>(dst);
    const int chunks = D / V;
    // neighbouring pairs of single elements are turned like split ones, one
    // element apart
    constexpr bool kSplit = !kInterleaved || V == 1;
    const int turned = kSplit ? half / V : 0;              // items that turn chunk p against another
    const int inside = kSplit ? 2 * turned : 0;            // chunks those cover
    const int items = turned + (chunks - inside + 1) / 2;
    for (int p = x0; p < items; p += xstep) {
        if (p < turned) {
            const int ia = kInterleaved ? 2 * p : p, ib = kInterleaved ? 2 * p + 1 : p + turned;
            C a = s[ia], b = s[ib];
            turn_split<T, V>(a, b, cs + p * V);
            d[ia] = a;
            d[ib] = b;
        } else {
            const int ia = inside + 2 * (p - turned), ib = ia + 1;
            const bool two = ib < chunks;
            C a = s[ia], b = a;
            if (two) b = s[ib];
            if (!kSplit) {
                if (ia * V < 2 * half) turn_inside<T, V>(a, cs + ia * V / 2);
                if (ib * V < 2 * half) turn_inside<T, V>(b, cs + ib * V / 2);
            }
            d[ia] = a;
            if (two) d[ib] = b;
        }
    }
}

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeArgs a) {
    extern __shared__ float2 s_cs[];                       // tokens_per_block x half
    __shared__ int64_t s_k[kMaxTokens], s_v[kMaxTokens];   // cache offsets, -1: none
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens_per_block;
    const int n = (int)min((int64_t)a.tokens_per_block, a.T - t0);
    const int tid = threadIdx.y * blockDim.x + threadIdx.x;

    for (int i = tid; i < n * a.half; i += blockDim.x * blockDim.y) {
        const int t = i / a.half, p = i - t * a.half;
        const int ax = min(max(a.axis[p], 0), a.axes - 1);
        const double turns = (double)a.positions[(t0 + t) * a.axes + ax] * (double)a.freq[p] * 0.31830988618379067154;
        float sn, cs;
        sincospif((float)(turns - 2.0 * rint(turns * 0.5)), &sn, &cs);
        s_cs[i] = make_float2(cs, a.sign * sn);
    }
    if (tid < n && a.slots != nullptr) {
        const int slot = a.slots[t0 + tid];
        const bool ok = slot >= 0 && slot < a.slots_in_cache;
        const int page = slot / a.page, off = slot - page * a.page;
        s_k[tid] = ok ? page * a.k_page + off * a.k_slot : -1;
        s_v[tid] = ok ? page * a.v_page + off * a.v_slot : -1;
    }
    __syncthreads();

    const int rows = a.hq + 2 * a.hkv;
    for (int r = threadIdx.y; r < n * rows; r += blockDim.y) {
        const int t = r / rows, h = r - t * rows;
        const float2* cs = s_cs + t * a.half;
        if (h < a.hq) {
            head_items<T, V, kInterleaved>(
                reinterpret_cast<const T*>(a.q.src) + (t0 + t) * a.q.src_tok + h * a.q.src_head,
                reinterpret_cast<T*>(a.q.dst) + (t0 + t) * a.q.dst_tok + h * a.q.dst_head, a.D, a.half, cs,
                threadIdx.x, blockDim.x);
        } else if (h < a.hq + a.hkv) {
            if (s_k[t] >= 0)
                head_items<T, V, kInterleaved>(
                    reinterpret_cast<const T*>(a.k.src) + (t0 + t) * a.k.src_tok + (h - a.hq) * a.k.src_head,
                    reinterpret_cast<T*>(a.k.dst) + s_k[t] + (h - a.hq) * a.k.dst_head, a.D, a.half, cs, threadIdx.x,
                    blockDim.x);
        } else if (s_v[t] >= 0) {
            const int g = h - a.hq - a.hkv;
            head_items<T, V, kInterleaved>(
                reinterpret_cast<const T*>(a.v.src) + (t0 + t) * a.v.src_tok + g * a.v.src_head,
                reinterpret_cast<T*>(a.v.dst) + s_v[t] + g * a.v.dst_head, a.D, 0, cs, threadIdx.x, blockDim.x);
        }
    }
}

template <typename T, int V>
void launch(const RopeArgs& a, bool interleaved, cudaStream_t st) {
    const int items = std::max(1, (a.D / V + 1) / 2);      // of one head
    int x = 1;
    while (x < items && x < 32) x *= 2;
    // Half the threads where a token has few items: the blocks' angles and loads
    // overlap better (12 heads of 64 columns in fp32: 23.1 us with 256, 20.6 with
    // 128; 48 heads of 128 in bf16: 41.1 and 45.3).
    const int threads = items * (a.hq + 2 * a.hkv) <= 128 ? kThreads / 2 : kThreads;
    const dim3 block(x, threads / x);
    const unsigned grid = (unsigned)((a.T + a.tokens_per_block - 1) / a.tokens_per_block);
    const size_t smem = (size_t)a.tokens_per_block * a.half * sizeof(float2);
    if (interleaved) rope_kernel<T, V, true><<<grid, block, smem, st>>>(a);
    else rope_kernel<T, V, false><<<grid, block, smem, st>>>(a);
}

bool aligned(const Rows& r, int64_t size) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(r.src) | reinterpret_cast<uintptr_t>(r.dst);
    return (p & 15) == 0 && ((r.src_tok | r.src_head | r.dst_tok | r.dst_head) * size) % 16 == 0;
}

// 16-byte chunks where every head, stride and the pairs' halves allow them,
// single elements otherwise (an odd D, a slice that starts off a boundary).
int run(RopeArgs& a, int32_t dtype, int32_t interleaved, cudaStream_t st) {
    if (a.T == 0) return MARS_OK;
    const int64_t size = dtype == MARS_DTYPE_F32 ? 4 : 2;
    const int V = (int)(16 / size);
    bool wide = a.D % V == 0 && (interleaved ? (2 * a.half) % V == 0 : a.half % V == 0) && aligned(a.q, size);
    if (a.slots != nullptr)
        wide = wide && aligned(a.k, size) && aligned(a.v, size) &&
               ((a.k_page | a.k_slot | a.v_page | a.v_slot) * size) % 16 == 0;
    // One token a block while that leaves SMs without one (4 blocks on each
    // are resident); up to four, to share the angles' latency, beyond.
    a.tokens_per_block = std::max(1, std::min(kMaxTokens, a.T / (148 * 4)));
    switch (dtype) {
        case MARS_DTYPE_F32: wide ? launch<float, 4>(a, interleaved, st) : launch<float, 1>(a, interleaved, st); break;
        case MARS_DTYPE_F16: wide ? launch<__half, 8>(a, interleaved, st) : launch<__half, 1>(a, interleaved, st); break;
        default:
            wide ? launch<__nv_bfloat16, 8>(a, interleaved, st) : launch<__nv_bfloat16, 1>(a, interleaved, st);
    }
    MARS_CUDA_TRY(cudaGetLastError());
    return MARS_OK;
}

int check_table(const mars_rope_table* r, int32_t D, int32_t T, const int32_t* d_positions, const char* fn) {
    if (r == nullptr) return fail(MARS_ERR_INVALID, std::string(fn) + ": NULL table");
    if (D <= 0 || T < 0) return fail(MARS_ERR_INVALID, std::string(fn) + ": head_dim must be positive, tokens not negative");
    if (r->rot_dim < 0 || r->rot_dim > D || r->rot_dim % 2 != 0)
        return fail(MARS_ERR_INVALID, std::string(fn) + ": rot_dim must be even and in [0, head_dim]");
    if (r->rot_dim / 2 > kMaxHalf)
        return fail(MARS_ERR_UNSUPPORTED, std::string(fn) + ": rot_dim must be at most " + std::to_string(2 * kMaxHalf));
    if (r->n_axes <= 0) return fail(MARS_ERR_INVALID, std::string(fn) + ": n_axes must be positive");
    if (T > 0 && (d_positions == nullptr || (r->rot_dim > 0 && (r->d_freq == nullptr || r->d_axis == nullptr))))
        return fail(MARS_ERR_INVALID, std::string(fn) + ": NULL argument");
    return MARS_OK;
}

}  // namespace

namespace mars {

int check_cache(const mars_kv_cache* c, const char* fn) {
    if (c == nullptr || c->k == nullptr || c->v == nullptr) return fail(MARS_ERR_INVALID, std::string(fn) + ": NULL cache");
    if (c->dtype != MARS_DTYPE_F16 && c->dtype != MARS_DTYPE_BF16)
        return fail(MARS_ERR_UNSUPPORTED, std::string(fn) + ": the cache holds fp16 or bf16");
    if (c->num_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->head_dim <= 0)
        return fail(MARS_ERR_INVALID, std::string(fn) + ": the cache's sizes must be positive");
    if ((int64_t)c->num_pages * c->page_size > 0x7fffffffLL)
        return fail(MARS_ERR_UNSUPPORTED, std::string(fn) + ": the cache holds at most 2^31 - 1 tokens");
    return MARS_OK;
}

}  // namespace mars

extern "C" int mars_rope(const mars_rope_table* table, int32_t dtype, const void* d_x, int64_t x_token_stride,
                         int64_t x_head_stride, void* d_y, int64_t y_token_stride, int64_t y_head_stride,
                         int32_t tokens, int32_t heads, int32_t head_dim, const int32_t* d_positions,
                         int32_t inverse, void* stream) {
    MARS_TRY(check_table(table, head_dim, tokens, d_positions, "mars_rope"));
    if (dtype != MARS_DTYPE_F32 && dtype != MARS_DTYPE_F16 && dtype != MARS_DTYPE_BF16)
        return fail(MARS_ERR_UNSUPPORTED, "mars_rope: dtype must be fp32, fp16 or bf16");
    if (heads <= 0 || (tokens > 0 && (d_x == nullptr || d_y == nullptr)))
        return fail(MARS_ERR_INVALID, "mars_rope: NULL argument or no heads");
    RopeArgs a{};
    a.q = Rows{static_cast<const char*>(d_x), static_cast<char*>(d_y), x_token_stride, x_head_stride, y_token_stride,
               y_head_stride};
    a.positions = d_positions;
    a.freq = table->d_freq;
    a.axis = table->d_axis;
    a.T = tokens;
    a.hq = heads;
    a.D = head_dim;
    a.half = table->rot_dim / 2;
    a.axes = table->n_axes;
    a.page = 1;
    a.sign = inverse ? -1.0f : 1.0f;
    return run(a, dtype, table->interleaved, static_cast<cudaStream_t>(stream));
}

extern "C" int mars_rope_append(const mars_rope_table* table, const mars_kv_cache* cache, const void* d_q,
                                int64_t q_token_stride, int64_t q_head_stride, const void* d_k,
                                int64_t k_token_stride, int64_t k_head_stride, const void* d_v,
                                int64_t v_token_stride, int64_t v_head_stride, void* d_q_out,
                                int64_t q_out_token_stride, int64_t q_out_head_stride, int32_t tokens,
                                int32_t q_heads, const int32_t* d_positions, const int32_t* d_slots, void* stream) {
    MARS_TRY(check_cache(cache, "mars_rope_append"));
    MARS_TRY(check_table(table, cache->head_dim, tokens, d_positions, "mars_rope_append"));
    if (q_heads <= 0 || (tokens > 0 && (d_q == nullptr || d_k == nullptr || d_v == nullptr || d_q_out == nullptr ||
                                        d_slots == nullptr)))
        return fail(MARS_ERR_INVALID, "mars_rope_append: NULL argument or no heads");
    RopeArgs a{};
    a.q = Rows{static_cast<const char*>(d_q), static_cast<char*>(d_q_out), q_token_stride, q_head_stride,
               q_out_token_stride, q_out_head_stride};
    a.k = Rows{static_cast<const char*>(d_k), static_cast<char*>(cache->k), k_token_stride, k_head_stride, 0,
               cache->k_head_stride};
    a.v = Rows{static_cast<const char*>(d_v), static_cast<char*>(cache->v), v_token_stride, v_head_stride, 0,
               cache->v_head_stride};
    a.k_page = cache->k_page_stride;
    a.k_slot = cache->k_slot_stride;
    a.v_page = cache->v_page_stride;
    a.v_slot = cache->v_slot_stride;
    a.slots = d_slots;
    a.slots_in_cache = (int64_t)cache->num_pages * cache->page_size;
    a.positions = d_positions;
    a.freq = table->d_freq;
    a.axis = table->d_axis;
    a.T = tokens;
    a.hq = q_heads;
    a.hkv = cache->kv_heads;
    a.D = cache->head_dim;
    a.half = table->rot_dim / 2;
    a.axes = table->n_axes;
    a.page = cache->page_size;
    a.sign = 1.0f;
    return run(a, cache->dtype, table->interleaved, static_cast<cudaStream_t>(stream));
}
