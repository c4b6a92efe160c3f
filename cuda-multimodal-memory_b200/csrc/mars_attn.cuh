// mars_attn.cuh -- what the attention kernels over the paged cache share: the
// problem, and which keys a row sees.
//
// Row r of request b (its new tokens are the last of its kv_len) stands at
// position i = kv_len - new + r and sees key j when
//     j < prefix_b,  or  j <= i  and  i - j < window,        (j < kv_len)
// so a set of consecutive rows sees at most two ranges: [0, prefix) and
// [low, high).  The score is
//     s = cap * tanh(scale * q.k / cap) - decay_h * max(0, i - j),
// out = sum_j softmax(s)_j v_j and lse = log sum_j exp(s_j); a row that sees
// nothing gets out = 0 and lse = -inf.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "mars_b200.h"

namespace mars {

// A cap: out * tanh(in * s), in units of log 2.  Up to |in * s| = 1/2 as s P(s^2),
// P a polynomial of degree 5 fitted here to the least largest relative error of
// tanh(x) / x (2^-24.5 in fp32), its coefficients taking the powers of in and out;
// beyond it by tanh_exp.  So the error is relative to the score, not to the cap.
// Which form a score takes follows from the score alone: the same in both kernels,
// whatever stands beside it.
// The polynomial has no special function: with two of them for a tanh and one for
// the softmax, capped scores took three times the exponentials' time.
struct Cap {
    float in, out, most;          // most: the largest |s| for the polynomial
    uint64_t c[6];                // each twice, for two scores an instruction
};

struct AttnArgs {
    const void* q;                // tokens x q_heads x D
    void* out;
    float* lse;                   // tokens x q_heads, or NULL
    const int32_t* cu_new;        // B + 1
    const int32_t* kv_lens;       // B
    const int32_t* tables;        // B x pitch
    const int32_t* prefix;        // B, or NULL
    const float* decay;           // q_heads, or NULL
    int64_t q_tok, q_head, o_tok, o_head;
    float scale, softcap;         // softcap 0: none
    Cap cap;
    int32_t window;               // 0: none
    int32_t T, B, hq, hkv, group, D, page, num_pages, pitch;
};

struct Request {
    int first, rows;              // its new tokens: [first, first + rows) of the call
    int len;                      // keys in its cache
    int prefix;
};

__device__ __forceinline__ Request load_request(const AttnArgs& a, int b) {
    Request r;
    r.first = min(max(a.cu_new[b], 0), a.T);
    r.rows = min(max(a.cu_new[b + 1], r.first), a.T) - r.first;
    // (keys are counted in 32 bits, tiles past the last one included)
    r.len = (int)min((int64_t)max(a.kv_lens[b], 0), min((int64_t)a.pitch * a.page, (int64_t)MARS_ATTN_MAX_KEYS));
    r.prefix = a.prefix != nullptr ? min(max(a.prefix[b], 0), r.len) : 0;
    return r;
}

// Keys beside the prefix that rows [r0, r1) see, all together.
__device__ __forceinline__ void row_range(const AttnArgs& a, const Request& r, int r0, int r1, int* low, int* high) {
    const int64_t shift = (int64_t)r.len - r.rows;
    *high = (int)max((int64_t)r.prefix, min((int64_t)r.len, shift + r1));
    const int64_t lo = a.window > 0 ? shift + r0 - a.window + 1 : 0;
    *low = (int)min((int64_t)*high, max((int64_t)r.prefix, lo));
}

// tanh x = 1 - 2 / (1 + e^2x): exact to a few units of 2^-24 of 1, so of the
// cap for the capped score (tanh.approx keeps 2^-11 of the cap, 0.02 at a cap
// of 50).  Two instructions of the special function unit; volatile, because a
// branch around each where the result is selected took twice the time.
__device__ __forceinline__ float tanh_exp(float x) {
    float e, r;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * 2.8853900817779268f));      // 2 / ln 2
    asm volatile("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));                     // 1 / inf = 0
    return fmaf(-2.0f, r, 1.0f);
}

}  // namespace mars
