// mars_attn_mma.cuh -- instruction wrappers and the work descriptor that the
// two attention kernels (mars_attn_short.cu, mars_attn_chunk.cu) share.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "mars_attn.cuh"
#include "mars_kv.h"
#include "mars_sm100.cuh"

namespace mars {

constexpr int kShortRows = 16;            // rows (tokens x query heads of a key head) of a short tile
constexpr int kPartCols = MARS_ATTN_MAX_HEAD_DIM;

// A call's working memory and launch figures.
struct AttnWork {
    float* part_o;                // parts of split units: slots x rows x kPartCols
    float2* part_ml;              // slots x rows: maximum (log 2 units) and sum
    unsigned int* tickets;        // one for each CTA, zero between calls
    int* err;                     // device word: a bounded wait gave up
    int* host_err;                // the same, where the host sees it
    int box;                      // keys of one TMA box: divides a page and a tile
    int min_share;                // tiles a CTA takes at least
};

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const void* tmap, uint64_t* bar, int32_t x, int32_t y,
                                            int32_t z, int32_t u) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(sm100::smem_u32(smem_dst)), "l"(tmap), "r"(sm100::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(u)
        : "memory");
}

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ void st_shared_zero16(uint32_t addr) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// d += a (16 x 16, rows) x b (16 x 8, columns), fp32 accumulators.
template <typename T> __device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^x by the special function unit: 2 units in the last place, 0 for -inf.
__device__ __forceinline__ float exp2f_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two values rounded to T, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Host side (mars_attn.cu).
// The largest power of two that divides a page and a tile of keys.
int page_box(int page, int tile);
// Tensor maps of the pages: box of 64 columns x `box` tokens of one head.
int page_maps(const mars_kv_cache* cache, int box, CUtensorMap* k, CUtensorMap* v);
// Allows the kernel `bytes` of dynamic shared memory on the current device
// (done: the devices where it has been).
int allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& done);

int attn_short(const AttnArgs& a, AttnWork w, const mars_kv_cache* cache, int num_sms, cudaStream_t st);

}  // namespace mars
