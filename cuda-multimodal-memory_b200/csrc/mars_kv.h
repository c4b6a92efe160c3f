// mars_kv.h -- host-side context of the paged key/value cache operators
// (mars_kv.cu: lengths to tables, mars_rope.cu: rotary positions and cache
// writes, mars_attn*.cu: attention over the pages).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "mars_b200.h"
#include "mars_internal.h"

namespace mars { struct ChunkStart; }

struct mars_kv_ctx {
    int32_t device = 0;
    int32_t max_requests = 0;
    int32_t num_sms = 0;
    cudaStream_t stream = nullptr;

    // Arrival counters (kTicket*), zero between calls: a call's last block
    // puts back the one it used.  First kKvTickets, then one for each CTA of an
    // attention kernel.
    unsigned int* d_tickets = nullptr;

    // Attention: parts of units that several CTAs share (mars_attn_short.cu),
    // and the word, in mapped host memory, that a bounded wait which gave up sets.
    float* d_part_o = nullptr;
    float2* d_part_ml = nullptr;
    float* d_chunk_o = nullptr;         // the same for mars_attn_chunk.cu
    float2* d_chunk_ml = nullptr;
    mars::ChunkStart* d_starts = nullptr;
    int* d_failed = nullptr;            // after the starts, in the same allocation
    int* h_err = nullptr;
    uint64_t wait_ns = 0;               // the waits' limit
    bool stall = false;                 // test hook: the next attention call's first CTA loads nothing

    // The working memory above holds one call at a time.  `used` is recorded
    // after every call outside a capture; a call on another stream waits for it.
    cudaEvent_t used = nullptr;
    bool any = false;
    unsigned long long last_id = 0;     // that call's stream (cudaStreamGetId)
    unsigned long long now_id = 0;      // the call under way: its stream,
    bool captured = false;              // and whether it is part of a capture
};

namespace mars {

constexpr int kTicketRelease = 0;
constexpr int kTicketPlan = 1;
constexpr int kKvTickets = 2;

// The attention kernels' parts (5 or 39 MB), made by the first call of each kind.
int kv_attn_memory(mars_kv_ctx* c, bool chunk);
constexpr uint64_t kWaitNs = 2000000000ull;

// MARS_ERR_TIMEOUT, once, if a wait has given up since the last report.
int kv_report(mars_kv_ctx* c);
// The stream of a call on `c`, ordered after the context's previous call.
int kv_begin(mars_kv_ctx* c, void* stream, cudaStream_t* st);
// Marks the end of the call's work on `st`.
int kv_end(mars_kv_ctx* c, cudaStream_t st);
// Sizes and type of a cache that a call names.
int check_cache(const mars_kv_cache* c, const char* fn);

}  // namespace mars
