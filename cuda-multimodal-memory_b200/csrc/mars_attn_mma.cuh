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

// Where a CTA's share of a chunk call's work begins: key tile `tile` of head h
// of row tile pair qt of request b.
struct ChunkStart {
    int32_t b, qt, h, tile;
};

// A call's working memory and launch figures.
struct AttnWork {
    float* part_o;                // parts of split units: slots x rows x kPartCols
    float2* part_ml;              // slots x rows: maximum (log 2 units) and sum
    unsigned int* tickets;        // one for each CTA, zero between calls
    float* chunk_o;               // chunk kernel: slots x kPartCols x 256 rows
    float2* chunk_ml;             // slots x 256 rows
    ChunkStart* starts;           // one for each CTA and the end
    int* failed;                  // one for each CTA: a wait of it gave up
    int* host_err;                // host memory: code of a bounded wait that gave up
    uint64_t wait_ns;             // their limit
    int stall;                    // test hook: this CTA loads nothing, so its waits run out (-1: none)
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

// Bounded waits of the attention kernels, for all lanes of a warp: false after
// `limit` (two seconds, where a step of these pipelines takes microseconds), with
// `code` in the CTA's error word.  No CTA waits for another, so the word is the
// CTA's own, in shared memory: nothing of a wait that gave up is left for other
// CTAs, calls or replays to meet.  drain: a wait for copies or products in flight,
// which goes on when others have given up.
struct WaitLimit {
    int* err;                     // shared
    uint64_t ns;
};
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, int* err, uint64_t limit_ns, int code, bool drain) {
    // Kept small (unrolled, the polls of twenty waits were most of a 148 KB
    // kernel, and its path through them missed the instruction cache).
    uint64_t begin = 0;
#pragma unroll 1
    for (uint32_t i = 1;; ++i) {
        if (sm100::mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 0) {
            const uint64_t now = now_ns();
            if (begin == 0) begin = now;
            if (now - begin > limit_ns || (!drain && *((volatile int*)err) != 0)) break;
        }
    }
    atomicCAS(err, 0, code);
    return false;
}
inline __device__ __noinline__ bool wait_on_far(uint64_t* bar, uint32_t parity, int* err, uint64_t limit_ns, int code, bool drain) {
    return wait_on(bar, parity, err, limit_ns, code, drain);
}
// kFar: what follows a first poll that fails stands out of line, once for all waits.
// The chunk kernel has twenty of them (8 capped chunks 188 us written out, 174 out of
// line; prompts 830 and 783), the short kernel two (64 ragged requests 197 us written
// out, 211 out of line).  The short kernel's also do not look at the error word: its
// warps wait for the same loads, so their limits run out together (204.0 us with the
// look, 203.2 without).
template <bool kFar>
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, const WaitLimit& limit, int code, bool drain) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    return kFar ? wait_on_far(bar, parity, limit.err, limit.ns, code, drain)
                : wait_on(bar, parity, limit.err, limit.ns, code, true);
}
template <bool kFar = false>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const WaitLimit& limit, int code) {
    return __all_sync(0xffffffffu, bounded_wait<kFar>(bar, parity, limit, code, false));
}
template <bool kFar = false>
__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity, const WaitLimit& limit, int code) {
    bounded_wait<kFar>(bar, parity, limit, code, true);
}
// Tells the host, and `failed` if there is one, of a wait of this CTA that gave up.
__device__ __forceinline__ void report_wait(const WaitLimit& limit, int* host_err, int* failed = nullptr) {
    const int code = *((volatile int*)limit.err);
    if (code == 0) return;
    *host_err = code;
    if (failed != nullptr) *failed = code;
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

// A part's sum, at maximum m, on the scale of top.  Without a maximum it is 0, or
// NaN: maxima pass over scores that are NaN, sums keep them.
__device__ __forceinline__ float scaled_sum(float m, float sum, float top) {
    return m == -INFINITY ? sum : sum * exp2f_fast(m - top);
}
// lse of a row (maximum in units of log 2): -inf only where nothing was seen.
__device__ __forceinline__ float log_sum(float top, float sum) {
    return sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// Two fp32 values in one register pair, and the packed arithmetic on them (one
// instruction for both).
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 split(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Whether s takes the polynomial.
__device__ __forceinline__ bool cap_is_small(float s, const Cap& t) { return fabsf(s) <= t.most; }
// Two scores that both do.
__device__ __forceinline__ float2 cap_small(float x, float y, const Cap& t) {
    const uint64_t s = pair(x, y), u = mul2(s, s);
    uint64_t p = t.c[5];
#pragma unroll
    for (int k = 4; k >= 0; --k) p = fma2(p, u, t.c[k]);
    return split(mul2(s, p));
}
// Two scores of any size.
__device__ __forceinline__ float2 cap_any(float x, float y, const Cap& t) {
    const float fx = t.out * tanh_exp(x * t.in), fy = t.out * tanh_exp(y * t.in);
    const float2 e = cap_small(x, y, t);
    return make_float2(cap_is_small(x, t) ? e.x : fx, cap_is_small(y, t) ? e.y : fy);
}

// Programmatic dependent launch: the next kernel of the stream may start; wait
// until the one before is complete and its writes are visible.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// Shared-memory descriptors of 128-byte swizzled operands differ in the low
// word only (address, and the distance of 64-column blocks for the one whose N
// is the contiguous index); the high word: 1,024 bytes between groups of 8
// rows, version 1, 128-byte swizzle.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);

// D[tmem] (+)= A[smem] x B[smem]^T, kind::f16.
__device__ __forceinline__ void mma_f16_lo(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
                 : "memory");
}

// A step's products by one elected lane of a converged warp, and the commit of
// what the lane issued so far to `bar`.  One statement, predicated by
// elect.sync: a branch around each instruction cost 110 cycles an instruction
// where the tensor cores take 48 to 64.
// D[tmem] = A[smem] x B[smem]^T over 64 kPanels columns (kPanel bytes between
// the blocks of 64).
template <int kPanels>
__device__ __forceinline__ void mma_scores(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint64_t* bar) {
    if (kPanels == 1)
        asm volatile(
        "{\n\t.reg .pred e, p, q;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, 0, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
        "mov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}"
        ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(kDescHigh), "r"(sm100::smem_u32(bar)) : "memory");
    else
        asm volatile(
        "{\n\t.reg .pred e, p, q;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, 0, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
        "mov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.s64 a, a, 1018;\n\tadd.s64 b, b, 1018;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}"
        ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(kDescHigh), "r"(sm100::smem_u32(bar)) : "memory");
}
// D[tmem] (+)= A[tmem] x B[smem] over 64 rows of B (8 columns of A and 2,048
// bytes of B an instruction).
__device__ __forceinline__ void mma_weights(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t idesc, bool add,
                                            uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e, p, q;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
        "mov.b32 a, %1;\n\tmov.b64 b, {%2, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, p;\n\t"
        "add.s32 a, a, 8;\n\tadd.s64 b, b, 128;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, q;\n\t"
        "add.s32 a, a, 8;\n\tadd.s64 b, b, 128;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, q;\n\t"
        "add.s32 a, a, 8;\n\tadd.s64 b, b, 128;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, q;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "r"(b_lo), "r"(idesc), "r"((uint32_t)add), "n"(kDescHigh), "r"(sm100::smem_u32(bar))
        : "memory");
}

// 32 lanes x N consecutive columns, complete on return: load and wait are one
// statement, so that the compiler has no registers in hand that the load has
// still to write (a copy or a spill between the two would take the old value
// and free a register that is written later).
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr) : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
          "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
          "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Host side (mars_attn.cu).
// The largest power of two that divides a page and a tile of keys.
int page_box(int page, int tile);
// Tensor maps of the pages: box of 64 columns x `box` tokens of one head.
int page_maps(const mars_kv_cache* cache, int box, CUtensorMap* k, CUtensorMap* v);
// Tensor map of the queries: box of 64 columns x all heads of one key head x
// `tokens` tokens.
int query_map(const AttnArgs& a, int32_t dtype, int tokens, CUtensorMap* q);
// Allows the kernel `bytes` of dynamic shared memory on the current device
// (done: the devices where it has been).
int allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& done);

int attn_short(const AttnArgs& a, AttnWork w, const mars_kv_cache* cache, int num_sms, cudaStream_t st);
int attn_chunk(const AttnArgs& a, AttnWork w, const mars_kv_cache* cache, int num_sms, cudaStream_t st);

}  // namespace mars
