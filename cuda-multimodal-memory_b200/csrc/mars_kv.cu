// mars_kv.cu -- block tables, slots and positions of a paged key/value cache,
// built on the GPU from the requests' lengths, and the context of the cache's
// operators.  The reference has no counterpart: it retrieves memories and
// leaves the answering to its caller.
//
// Pages are handed out from a stack of free page ids.  Request b of length
// len_b that gets new_b tokens needs ceil((len_b + new_b) / P) - ceil(len_b /
// P) pages; the requests take them from the stack's end in their own order.
// Token i of the call belongs to the request whose prefix sum of new_b covers
// i, and goes to slot table[b][pos / P] * P + pos % P.
//
// Both kernels do next to no arithmetic and move 4 to 12 bytes for each token
// and page; what bounds them is the launch and the chain lengths -> prefix sum
// -> page id -> slot (4.6 us on the device for 64 requests with a token each, 10
// for 300 prompts of 360,000 tokens; a call from Python takes 19 us, its host time).  So every block forms the prefix sums of all requests by
// itself (at most 8,192 of them, 64 KB from L2) instead of waiting for another
// launch, and finds a token's request by bisection in shared memory.  Inputs
// and outputs may be the same arrays: the last block to arrive (a counter, no
// spinning) writes the lengths and counts once all blocks have read them.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>
#include <vector>

#include "mars_attn_mma.cuh"
#include "mars_kv.h"

using namespace mars;

namespace {

// Words of pinned host memory, one for each context: a page for all of them
// (pinning one costs more than the rest of a context's creation).
std::mutex g_words_lock;
std::vector<int*> g_words;

int host_word(int** out) {
    std::lock_guard<std::mutex> lock(g_words_lock);
    if (g_words.empty()) {
        constexpr int kWords = 512;
        int* page = nullptr;
        MARS_CUDA_TRY(cudaHostAlloc(&page, kWords * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable));
        for (int i = 0; i < kWords; ++i) g_words.push_back(page + i);
    }
    *out = g_words.back();
    g_words.pop_back();
    return MARS_OK;
}

void free_host_word(int* w) {
    std::lock_guard<std::mutex> lock(g_words_lock);
    g_words.push_back(w);
}

}  // namespace

namespace mars {

int kv_attn_memory(mars_kv_ctx* c, bool chunk) {
    const size_t sms = (size_t)c->num_sms;
    if (!chunk && c->d_part_ml == nullptr) {
        const size_t slots = 2 * 2 * sms;          // two of each CTA, two CTAs an SM
        if (c->d_part_o == nullptr) MARS_CUDA_TRY(cudaMalloc(&c->d_part_o, slots * kShortRows * kPartCols * sizeof(float)));
        MARS_CUDA_TRY(cudaMalloc(&c->d_part_ml, slots * kShortRows * sizeof(float2)));
    }
    if (chunk && c->d_starts == nullptr) {
        const size_t rows = 256, slots = 2 * sms;
        if (c->d_chunk_o == nullptr) MARS_CUDA_TRY(cudaMalloc(&c->d_chunk_o, slots * rows * kPartCols * sizeof(float)));
        if (c->d_chunk_ml == nullptr) MARS_CUDA_TRY(cudaMalloc(&c->d_chunk_ml, slots * rows * sizeof(float2)));
        MARS_CUDA_TRY(cudaMalloc(&c->d_starts, (sms + 1) * sizeof(ChunkStart) + sms * sizeof(int)));
        c->d_failed = reinterpret_cast<int*>(c->d_starts + sms + 1);
    }
    return MARS_OK;
}

int kv_report(mars_kv_ctx* c) {
    const int code = *static_cast<volatile int*>(c->h_err);
    if (code == 0) return MARS_OK;
    *static_cast<volatile int*>(c->h_err) = 0;
    return fail(MARS_ERR_TIMEOUT, "a bounded wait (" + std::to_string(code) +
                                      ") of an earlier call gave up: its results are not valid");
}

int kv_begin(mars_kv_ctx* c, void* stream, cudaStream_t* st) {
    *st = stream != nullptr ? static_cast<cudaStream_t>(stream) : c->stream;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    MARS_CUDA_TRY(cudaStreamIsCapturing(*st, &cap));
    c->captured = cap != cudaStreamCaptureStatusNone;
    if (*static_cast<volatile int*>(c->h_err) != 0) {
        // All of the call's CTAs have reported once it has ended.
        if (!c->captured && c->any) MARS_CUDA_TRY(cudaEventSynchronize(c->used));
        return kv_report(c);
    }
    if (c->captured) return MARS_OK;               // a replay's order is its launcher's
    // The id tells streams apart, their handles do not: a destroyed stream's may be a new
    // one's, and cudaStreamPerThread is another stream in every thread.  (Waiting on the same
    // stream too would be as right, and 0.3 us of host time a call.)
    unsigned long long id = 0;
    MARS_CUDA_TRY(cudaStreamGetId(*st, &id));
    if (c->any && id != c->last_id) MARS_CUDA_TRY(cudaStreamWaitEvent(*st, c->used, 0));
    c->now_id = id;
    return MARS_OK;
}

int kv_end(mars_kv_ctx* c, cudaStream_t st) {
    if (c->captured) return MARS_OK;
    MARS_CUDA_TRY(cudaEventRecord(c->used, st));
    c->last_id = c->now_id;
    c->any = true;
    return MARS_OK;
}

}  // namespace mars

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

// Exclusive prefix sum over the block of two 64-bit counts a thread holds.
struct Pair { long long a, b; };

__device__ Pair block_exclusive(Pair v, Pair* total) {
    __shared__ Pair s_warp[kWarps + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Pair inc = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, inc.a, off);
        const long long b = __shfl_up_sync(0xffffffffu, inc.b, off);
        if (lane >= off) { inc.a += a; inc.b += b; }
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    if (threadIdx.x == 0) {
        Pair run{0, 0};
        for (int w = 0; w < kWarps; ++w) {
            const Pair t = s_warp[w];
            s_warp[w] = run;
            run.a += t.a;
            run.b += t.b;
        }
        s_warp[kWarps] = run;
    }
    __syncthreads();
    *total = s_warp[kWarps];
    const Pair base = s_warp[warp];
    return Pair{base.a + inc.a - v.a, base.b + inc.b - v.b};
}

// The bits that any thread of the block found.
__device__ int block_or(int bits) {
    __shared__ int s_bits;
    if (threadIdx.x == 0) s_bits = 0;
    __syncthreads();
    if (bits != 0) atomicOr(&s_bits, bits);
    __syncthreads();
    return s_bits;
}

// The last i in [0, n) with first[i] <= x (first[0] = 0 <= x).
__device__ __forceinline__ int owner(const int32_t* first, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

// True in every thread of the block that arrives last of the grid.
__device__ bool last_block(unsigned int* ticket) {
    __shared__ int s_last;
    if (gridDim.x == 1) { __syncthreads(); return true; }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
        if (s_last) { *ticket = 0; __threadfence(); }
    }
    __syncthreads();
    return s_last != 0;
}

struct ReleaseArgs {
    const int32_t* lens;
    const int32_t* flags;
    const int32_t* tables;
    int32_t* free_pages;
    const int32_t* free_count;
    int32_t* lens_out;
    int32_t* free_count_out;
    int32_t* status;
    int32_t B, pitch, page, free_cap;
    unsigned int* ticket;
};

// Pages of the flagged requests onto the free stack, request by request.
__global__ void __launch_bounds__(kThreads) kv_release_kernel(const ReleaseArgs a) {
    extern __shared__ int32_t s_first[];           // B: released pages before request b
    const int per = (a.B + kThreads - 1) / kThreads;
    const int b0 = threadIdx.x * per, b1 = min(a.B, b0 + per);
    Pair mine{0, 0};
    int bad = 0;
    for (int b = b0; b < b1; ++b) {
        if (a.flags[b] == 0) continue;
        const int len = a.lens[b];
        const long long pages = len > 0 ? ((long long)len + a.page - 1) / a.page : 0;
        if (len < 0) bad |= MARS_KV_BAD_LENGTH;
        if (pages > a.pitch) bad |= MARS_KV_TABLE_FULL;
        mine.a += pages;
    }
    Pair total;
    Pair at = block_exclusive(mine, &total);
    for (int b = b0; b < b1; ++b) {
        s_first[b] = (int32_t)at.a;
        if (a.flags[b] != 0 && a.lens[b] > 0) at.a += ((long long)a.lens[b] + a.page - 1) / a.page;
    }
    const int count = *a.free_count;
    if (count < 0 || count + total.a > a.free_cap) bad |= MARS_KV_STACK_FULL;
    bad = block_or(bad);
    if (bad == 0) {
        for (int j = blockIdx.x * kThreads + threadIdx.x; j < total.a; j += gridDim.x * kThreads) {
            const int b = owner(s_first, a.B, j);
            a.free_pages[count + j] = a.tables[(int64_t)b * a.pitch + (j - s_first[b])];
        }
    }
    if (!last_block(a.ticket)) return;
    for (int b = threadIdx.x; b < a.B; b += kThreads)
        a.lens_out[b] = bad == 0 && a.flags[b] != 0 ? 0 : a.lens[b];
    if (threadIdx.x == 0) {
        *a.free_count_out = bad == 0 ? count + (int)total.a : count;
        if (a.status != nullptr) *a.status = bad;
    }
}

struct PlanArgs {
    const int32_t* lens;
    const int32_t* added;
    int32_t* tables;
    const int32_t* free_pages;
    const int32_t* free_count;
    int32_t* lens_out;
    int32_t* free_count_out;
    int32_t* first;
    int32_t* slots;
    int32_t* positions;
    int32_t* status;
    int32_t B, pitch, page, free_cap, max_tokens;
    unsigned int* ticket;
};

__global__ void __launch_bounds__(kThreads) kv_plan_kernel(const PlanArgs a) {
    extern __shared__ int32_t s_mem[];
    int32_t* s_first = s_mem;                      // B + 1: tokens before request b
    int32_t* s_need = s_first + a.B + 1;           // B + 1: new pages before request b
    int32_t* s_len = s_need + a.B + 1;             // B
    const int P = a.page;
    const int per = (a.B + kThreads - 1) / kThreads;
    const int b0 = threadIdx.x * per, b1 = min(a.B, b0 + per);
    Pair mine{0, 0};
    int bad = 0;
    for (int b = b0; b < b1; ++b) {
        const int len = a.lens[b], add = a.added[b];
        if (len < 0 || add < 0) { bad |= MARS_KV_BAD_LENGTH; continue; }
        const long long after = (long long)len + add;
        if (after > 0x7fffffffLL) { bad |= MARS_KV_BAD_LENGTH; continue; }
        const long long want = (after + P - 1) / P;
        if (want > a.pitch) bad |= MARS_KV_TABLE_FULL;
        mine.a += add;
        mine.b += want - ((long long)len + P - 1) / P;
    }
    Pair total;
    Pair at = block_exclusive(mine, &total);
    const int count = *a.free_count;
    if (count < 0 || count > a.free_cap) bad |= MARS_KV_STACK_FULL;
    else if (total.b > count) bad |= MARS_KV_NO_PAGES;
    if (total.a > a.max_tokens) bad |= MARS_KV_TOO_MANY_TOKENS;
    bad = block_or(bad);
    for (int b = b0; b < b1; ++b) {
        const int len = a.lens[b], add = a.added[b];
        s_first[b] = (int32_t)at.a;
        s_need[b] = (int32_t)at.b;
        s_len[b] = len;
        if (bad == 0) {
            at.a += add;
            at.b += ((long long)len + add + P - 1) / P - ((long long)len + P - 1) / P;
        }
    }
    const int tokens = bad == 0 ? (int)total.a : 0, fresh = bad == 0 ? (int)total.b : 0;
    if (threadIdx.x == 0) { s_first[a.B] = tokens; s_need[a.B] = fresh; }
    __syncthreads();

    const int step = gridDim.x * kThreads, me = blockIdx.x * kThreads + threadIdx.x;
    for (int j = me; j < fresh; j += step) {
        const int b = owner(s_need, a.B, j);
        const int held = (int)(((long long)s_len[b] + P - 1) / P);
        a.tables[(int64_t)b * a.pitch + held + (j - s_need[b])] = a.free_pages[count - 1 - j];
    }
    // A token's page: one that the request held before the call, or the one
    // that the loop above hands it (taken from the stack again, so that no
    // thread waits for another's write).
    for (int64_t i = me; i < a.max_tokens; i += step) {
        int slot = -1, pos = -1;
        if (i < tokens) {
            const int b = owner(s_first, a.B, (int)i);
            pos = s_len[b] + ((int)i - s_first[b]);
            const int held = (int)(((long long)s_len[b] + P - 1) / P), col = pos / P;
            const int page = col < held ? a.tables[(int64_t)b * a.pitch + col]
                                        : a.free_pages[count - 1 - (s_need[b] + (col - held))];
            slot = page * P + (pos - col * P);
        }
        a.slots[i] = slot;
        if (a.positions != nullptr) a.positions[i] = pos;
    }
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= a.B; b += kThreads) a.first[b] = bad == 0 ? s_first[b] : 0;
    if (!last_block(a.ticket)) return;
    for (int b = threadIdx.x; b < a.B; b += kThreads)
        a.lens_out[b] = bad == 0 ? s_len[b] + (s_first[b + 1] - s_first[b]) : s_len[b];
    if (threadIdx.x == 0) {
        *a.free_count_out = count - fresh;
        *a.status = bad;
    }
}

int check_plan(const mars_kv_ctx* c, int32_t B, int32_t page_size, int32_t table_pitch, int32_t free_cap,
               const char* fn) {
    if (c == nullptr) return fail(MARS_ERR_INVALID, std::string(fn) + ": NULL context");
    if (B < 0 || B > c->max_requests)
        return fail(MARS_ERR_CAPACITY, std::string(fn) + ": B must be in [0, " + std::to_string(c->max_requests) + "]");
    if (page_size <= 0 || table_pitch <= 0 || free_cap < 0)
        return fail(MARS_ERR_INVALID, std::string(fn) + ": page_size and table_pitch must be positive, free_cap not negative");
    return MARS_OK;
}

}  // namespace

extern "C" int mars_kv_ctx_create(int32_t device, int32_t max_requests, mars_kv_ctx** out) {
    if (out == nullptr) return fail(MARS_ERR_INVALID, "mars_kv_ctx_create: NULL out");
    *out = nullptr;
    if (max_requests <= 0 || max_requests > MARS_KV_MAX_REQUESTS)
        return fail(MARS_ERR_INVALID, "mars_kv_ctx_create: max_requests must be in [1, " +
                                          std::to_string(MARS_KV_MAX_REQUESTS) + "]");
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
        (void)cudaGetLastError();
        return fail(MARS_ERR_NO_DEVICE, "mars_kv_ctx_create: no CUDA device");
    }
    if (device < 0 || device >= count) return fail(MARS_ERR_INVALID, "mars_kv_ctx_create: no such device");
    MarsDeviceGuard g(device);
    if (!g.ok) return fail(MARS_ERR_CUDA, "mars_kv_ctx_create: cudaSetDevice failed");
    int major = 0, sms = 0;
    MARS_CUDA_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
    MARS_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    if (major != 10) return fail(MARS_ERR_NO_DEVICE, "mars_kv_ctx_create: needs an sm_100 device");
    mars_kv_ctx* c = new mars_kv_ctx();
    c->device = device;
    c->max_requests = max_requests;
    c->num_sms = sms;
    c->wait_ns = kWaitNs;
    auto build = [&]() -> int {
        MARS_CUDA_TRY(cudaStreamCreateWithFlags(&c->stream, cudaStreamNonBlocking));
        MARS_CUDA_TRY(cudaEventCreateWithFlags(&c->used, cudaEventDisableTiming));
        const size_t words = kKvTickets + 2 * (size_t)sms;
        MARS_CUDA_TRY(cudaMalloc(&c->d_tickets, words * sizeof(unsigned int)));
        MARS_TRY(host_word(&c->h_err));
        *c->h_err = 0;
        MARS_CUDA_TRY(cudaMemsetAsync(c->d_tickets, 0, words * sizeof(unsigned int), c->stream));
        // the largest context's: the attribute is the device's, not the context's
        MARS_CUDA_TRY(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (3 * MARS_KV_MAX_REQUESTS + 2) * (int)sizeof(int32_t)));
        MARS_CUDA_TRY(cudaStreamSynchronize(c->stream));
        return MARS_OK;
    };
    const int st = build();
    if (st != MARS_OK) {
        mars_kv_ctx_destroy(c);
        return st;
    }
    *out = c;
    return MARS_OK;
}

extern "C" int mars_kv_ctx_destroy(mars_kv_ctx* c) {
    if (c == nullptr) return MARS_OK;
    MarsDeviceGuard g(c->device);
    if (c->any) cudaEventSynchronize(c->used);
    if (c->d_tickets != nullptr) cudaFree(c->d_tickets);
    if (c->d_part_o != nullptr) cudaFree(c->d_part_o);
    if (c->d_part_ml != nullptr) cudaFree(c->d_part_ml);
    if (c->d_chunk_o != nullptr) cudaFree(c->d_chunk_o);
    if (c->d_chunk_ml != nullptr) cudaFree(c->d_chunk_ml);
    if (c->d_starts != nullptr) cudaFree(c->d_starts);
    if (c->h_err != nullptr) free_host_word(c->h_err);
    if (c->used != nullptr) cudaEventDestroy(c->used);
    if (c->stream != nullptr) cudaStreamDestroy(c->stream);
    delete c;
    return MARS_OK;
}

extern "C" void* mars_kv_ctx_stream(const mars_kv_ctx* c) { return c != nullptr ? c->stream : nullptr; }

extern "C" int mars_kv_ctx_status(mars_kv_ctx* c) {
    if (c == nullptr) return fail(MARS_ERR_INVALID, "mars_kv_ctx_status: NULL context");
    MarsDeviceGuard g(c->device);
    if (c->any) MARS_CUDA_TRY(cudaEventSynchronize(c->used));
    return kv_report(c);
}

extern "C" int mars_kv_ctx_debug_wait(mars_kv_ctx* c, uint64_t limit_ns, int32_t stall) {
    if (c == nullptr) return fail(MARS_ERR_INVALID, "mars_kv_ctx_debug_wait: NULL context");
    c->wait_ns = limit_ns == 0 ? kWaitNs : limit_ns;
    c->stall = stall != 0;
    return MARS_OK;
}

extern "C" int mars_kv_release(mars_kv_ctx* c, int32_t B, const int32_t* d_kv_lens, const int32_t* d_release,
                               const int32_t* d_tables, int32_t table_pitch, int32_t page_size,
                               int32_t* d_free_pages, int32_t free_cap, const int32_t* d_free_count,
                               int32_t* d_kv_lens_out, int32_t* d_free_count_out, int32_t* d_status, void* stream) {
    MARS_TRY(check_plan(c, B, page_size, table_pitch, free_cap, "mars_kv_release"));
    if ((B > 0 && (d_kv_lens == nullptr || d_release == nullptr || d_tables == nullptr || d_kv_lens_out == nullptr)) ||
        (free_cap > 0 && d_free_pages == nullptr) || d_free_count == nullptr || d_free_count_out == nullptr)
        return fail(MARS_ERR_INVALID, "mars_kv_release: NULL argument");
    MarsDeviceGuard g(c->device);
    cudaStream_t st;
    MARS_TRY(kv_begin(c, stream, &st));
    ReleaseArgs a{d_kv_lens, d_release, d_tables, d_free_pages, d_free_count, d_kv_lens_out, d_free_count_out,
                  d_status, B, table_pitch, page_size, free_cap, c->d_tickets + kTicketRelease};
    const int64_t most = std::min<int64_t>((int64_t)B * table_pitch, free_cap);
    const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>(c->num_sms, most / (4 * kThreads)));
    kv_release_kernel<<<blocks, kThreads, std::max(B, 1) * sizeof(int32_t), st>>>(a);
    MARS_CUDA_TRY(cudaGetLastError());
    return kv_end(c, st);
}

extern "C" int mars_kv_plan(mars_kv_ctx* c, int32_t B, const int32_t* d_kv_lens, const int32_t* d_new_lens,
                            int32_t* d_tables, int32_t table_pitch, int32_t page_size, const int32_t* d_free_pages,
                            int32_t free_cap, const int32_t* d_free_count, int32_t max_tokens,
                            int32_t* d_kv_lens_out, int32_t* d_free_count_out, int32_t* d_cu_new, int32_t* d_slots,
                            int32_t* d_positions, int32_t* d_status, void* stream) {
    MARS_TRY(check_plan(c, B, page_size, table_pitch, free_cap, "mars_kv_plan"));
    if (max_tokens < 0) return fail(MARS_ERR_INVALID, "mars_kv_plan: max_tokens must not be negative");
    if ((B > 0 && (d_kv_lens == nullptr || d_new_lens == nullptr || d_tables == nullptr || d_kv_lens_out == nullptr)) ||
        (free_cap > 0 && d_free_pages == nullptr) || (max_tokens > 0 && d_slots == nullptr) ||
        d_free_count == nullptr || d_free_count_out == nullptr || d_cu_new == nullptr || d_status == nullptr)
        return fail(MARS_ERR_INVALID, "mars_kv_plan: NULL argument");
    MarsDeviceGuard g(c->device);
    cudaStream_t st;
    MARS_TRY(kv_begin(c, stream, &st));
    PlanArgs a{d_kv_lens, d_new_lens, d_tables, d_free_pages, d_free_count, d_kv_lens_out, d_free_count_out,
               d_cu_new, d_slots, d_positions, d_status, B, table_pitch, page_size, free_cap, max_tokens,
               c->d_tickets + kTicketPlan};
    const int blocks = std::max(1, std::min(c->num_sms, max_tokens / (2 * kThreads)));
    kv_plan_kernel<<<blocks, kThreads, (3 * B + 2) * sizeof(int32_t), st>>>(a);
    MARS_CUDA_TRY(cudaGetLastError());
    return kv_end(c, st);
}
