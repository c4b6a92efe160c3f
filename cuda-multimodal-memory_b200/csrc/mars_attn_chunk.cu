// mars_attn_chunk.cu -- attention over the paged cache for chunks and whole
// prompts, on the 5th-generation tensor cores.
//
// A unit is 256 rows of one key head (two tiles of 128: tokens x the query
// heads that share the key head, so one read of keys and values serves them
// all) against the 128-key tiles that any of its rows sees.  Scores S = Q K^T
// go to TMEM, 64 keys at a time; a warpgroup for each of the two row tiles
// turns them into weights P (one thread a row: no shuffles), writes P over S as
// the second product's operand, and O += P V stays in TMEM for the whole unit:
//
//    columns  [0,64) S0/P0 first half  [64,128) second half  [128,256) the same
//             of row tile 1  [256,384) O0  [384,512) O1
//
// While a warpgroup works on one half, the other half's weights are multiplied
// and the next scores are made there, so it has scores to go on with:
// with scores of 128 keys at once (one buffer) each tile was a chain softmax ->
// O -> next S of 5,000 cycles for 2,048 cycles of products.
// The running maximum that P is scaled by follows the true one only when it
// is 2^8 behind: P stays below 2^8 (harmless in fp32 sums and in the type's
// relative precision), and O is rescaled a few times a unit instead of at
// every tile.  Sums, maxima and O are fp32; P is rounded to the cache's type
// because the product takes both operands of one type.
//
// Roles of a CTA (one on each SM): warp 0 loads by TMA (a lane for each box of
// a page), warps 1 and 3 issue the products of row tile 0 and 1, warp 2 zeroes
// the values of keys that no row sees (they may be anything, and 0 x NaN is
// NaN), warps 4-7 and 8-11 are the two softmax warpgroups.
//
// Work is shared as in mars_attn_short.cu: the units' tiles in one sequence,
// an equal share for each CTA.  A one-block kernel before it finds the shares
// (prompts have thousands of units), a kernel after it joins cut units; their
// set-ups overlap (programmatic dependent launch).
//
// Bound: the softmax warps.  64 keys of the two row tiles take 1,280 cycles of
// products at D = 128 (S 16 x 48, read from shared memory at its full rate; O 8 x
// 64) and 1,024 of exponentials (16 ex2 a cycle), measured alone; together a step
// takes 1,900 to 2,200.  A trace of a prompt gives a warpgroup 1,190 of them for
// exponentials, 290 for loading the scores and their maximum, 115 for rescaling
// and 230 for waiting: two softmax warps a scheduler go through these one after
// another, and tensor pipe and special function unit are each half busy.  Capped
// scores with a decay took 4,450 cycles a step in the same trace, 2,200 of them
// for the scores' shaping and maximum.  All variants are at their 168 registers
// and spill 200 to 240 bytes.
// Measured (bf16, 128 columns): two prompts of 8,192 and 4,142 tokens, 32 heads on
// 8, 815 us = 867 TFLOP/s under the power cap (the library's sustained rate for a
// plain product: 1,398).  8 chunks of up to 512 on up to 4,000, 16 heads on 4:
// 98 us, with decay 140, with decay and cap 175, scores beyond half the cap 216.
// Tried and dropped: exponentials on the FMA units beside the special function
// unit (slower: 8 FMA cycles an element against 8 of ex2), the warpgroups held
// out of step, one buffer of 128 keys' scores (915 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "mars_attn.cuh"
#include "mars_attn_mma.cuh"
#include "mars_kv.h"
#include "mars_sm100.cuh"

using namespace mars;
using namespace mars::sm100;

namespace {

constexpr int kTile = 128;                      // keys of a ring slot
constexpr int kHalf = 64;                       // keys of one step of a row tile
constexpr int kRows = 128;                      // rows of one of the two tiles
constexpr int kThreads = 384;
constexpr int kUnitCost = 1;                    // a unit's start and end, in tiles
constexpr float kSlack = 8.0f;                  // how far (log 2) the maximum in use may lag
constexpr float kLog2e = 1.4426950408889634f;

template <int kPanels> struct Layout {
    static constexpr int kPanel = kTile * 128;                    // bytes: 128 rows x 64 columns
    static constexpr int kQ = 2 * kPanels * kPanel;
    static constexpr int kSlot = kPanels * kPanel;                // one tile of keys or of values
    static constexpr int kSlots = kPanels == 2 ? 5 : 10;
    static constexpr int kSmem = 1024 + kQ + kSlots * kSlot;
};

struct Unit {
    int row0, rows;               // tokens
    int nq;                       // row tiles: 1 or 2
    int n1, s2, tiles;            // tiles of the prefix; first tile of the rest; in all
    int tiles0;                   // tiles that the first row tile sees, from the front
    int low, high;
};

__device__ __forceinline__ Unit make_unit(const AttnArgs& a, const Request& r, int qt, int per) {
    Unit u;
    u.row0 = qt * 2 * per;
    u.rows = min(2 * per, r.rows - u.row0);
    u.nq = u.rows > per ? 2 : 1;
    row_range(a, r, u.row0, u.row0 + u.rows, &u.low, &u.high);
    u.n1 = (r.prefix + kTile - 1) / kTile;
    u.s2 = max(u.n1, u.low / kTile);
    u.tiles = u.n1 + max(0, (u.high + kTile - 1) / kTile - u.s2);
    int low0, high0;
    row_range(a, r, u.row0, u.row0 + min(per, u.rows), &low0, &high0);
    u.tiles0 = u.n1 + max(0, (high0 + kTile - 1) / kTile - u.s2);
    return u;
}

__device__ __forceinline__ int key_of(const Unit& u, int t) { return (t < u.n1 ? t : u.s2 + t - u.n1) * kTile; }

// The lowest n bits (n < 0: none, n > 31: all).
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// ---- shares -----------------------------------------------------------------

constexpr int kPlanThreads = 256;

__device__ long long plan_scan(long long v, long long* total) {
    __shared__ long long s_sum[kPlanThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += o;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = inc;
    __syncthreads();
    long long before = 0, all = 0;
    for (int i = 0; i < kPlanThreads / 32; ++i) {
        if (i < warp) before += s_sum[i];
        all += s_sum[i];
    }
    *total = all;
    return before + inc - v;
}

// starts[i]: where CTA i's share begins; starts[ctas]: the end.
__global__ void __launch_bounds__(kPlanThreads) attn_chunk_plan_kernel(const AttnArgs a, ChunkStart* starts, int* failed,
                                                                       int ctas) {
    launch_dependents();                          // the main kernel sets itself up meanwhile
    extern __shared__ int s_units[];              // B: units (of one head) before request b
    const int per = kRows / a.group;
    const int each = (a.B + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(a.B, (int)threadIdx.x * each), b1 = min(a.B, b0 + each);
    long long mine = 0, units;
    for (int b = b0; b < b1; ++b) mine += (load_request(a, b).rows + 2 * per - 1) / (2 * per);
    long long at = plan_scan(mine, &units);
    for (int b = b0; b < b1; ++b) {
        s_units[b] = (int)at;
        at += (load_request(a, b).rows + 2 * per - 1) / (2 * per);
    }
    __syncthreads();
    const int n = (int)units, chunk = (n + kPlanThreads - 1) / kPlanThreads;
    const int u0 = min(n, (int)threadIdx.x * chunk), u1 = min(n, u0 + chunk);
    int first = 0;
    if (u0 < u1) {                                // the request of unit u0: the last with s_units[b] <= u0
        int hi = a.B;
        while (hi - first > 1) {
            const int mid = (first + hi) >> 1;
            if (s_units[mid] <= u0) first = mid; else hi = mid;
        }
    }
    long long cost = 0, total;
    int b = first;
    Request r{};
    if (u0 < u1) r = load_request(a, b);
    for (int u = u0; u < u1; ++u) {
        while (u >= s_units[b] + (r.rows + 2 * per - 1) / (2 * per)) r = load_request(a, ++b);
        cost += (long long)(max(1, make_unit(a, r, u - s_units[b], per).tiles) + kUnitCost) * a.hkv;
    }
    long long x = plan_scan(cost, &total);
    const long long share = max((total + ctas - 1) / ctas, (long long)(2 + kUnitCost));
    b = first;
    if (u0 < u1) r = load_request(a, b);
    for (int u = u0; u < u1; ++u) {
        while (u >= s_units[b] + (r.rows + 2 * per - 1) / (2 * per)) r = load_request(a, ++b);
        const int qt = u - s_units[b], tiles = make_unit(a, r, qt, per).tiles, c = max(1, tiles) + kUnitCost;
        // shares that begin inside this unit's heads
        for (long long i = (x + share - 1) / share; i < ctas && i * share < x + (long long)c * a.hkv; ++i) {
            const long long in = i * share - x;
            starts[i] = ChunkStart{b, qt, (int)(in / c), min(max((int)(in % c) - kUnitCost, 0), max(tiles - 1, 0))};
        }
        x += (long long)c * a.hkv;
    }
    for (long long i = threadIdx.x; i <= ctas; i += kPlanThreads)
        if (i == ctas || i * share >= total) starts[i] = ChunkStart{a.B, 0, 0, 0};
    for (int i = threadIdx.x; i < ctas; i += kPlanThreads) failed[i] = 0;
}

// ---- the kernel -------------------------------------------------------------

// A share's pieces, walked alike by every role.
struct Walk {
    ChunkStart cur, stop;
    Request r;
    Unit u;
    int begin, end;               // tiles of the unit
    int count[2];                 // of them, those that each row tile sees

    __device__ __forceinline__ void set(const AttnArgs& a, int per) {
        u = make_unit(a, r, cur.qt, per);
        begin = cur.tile;
        end = u.tiles;
        if (cur.b == stop.b && cur.qt == stop.qt && cur.h == stop.h) end = stop.tile;
        const int n = end - begin;
        count[0] = u.nq == 2 ? max(0, min(u.tiles0 - begin, n)) : n;
        count[1] = u.nq == 2 ? n : 0;
    }
    __device__ __forceinline__ bool start(const AttnArgs& a, const ChunkStart* starts, int cta, int per) {
        cur = starts[cta];
        stop = starts[cta + 1];
        if (done()) return false;
        r = load_request(a, cur.b);
        set(a, per);
        return true;
    }
    __device__ __forceinline__ bool done() const {
        return cur.b == stop.b && cur.qt == stop.qt && cur.h == stop.h && cur.tile == stop.tile;
    }
    __device__ __forceinline__ bool next(const AttnArgs& a, int per) {
        if (cur.b == stop.b && cur.qt == stop.qt && cur.h == stop.h) return false;
        cur.tile = 0;
        if (++cur.h == a.hkv) {
            cur.h = 0;
            if (++cur.qt * 2 * per >= r.rows) {
                cur.qt = 0;
                do {
                    if (++cur.b >= a.B) return false;
                    r = load_request(a, cur.b);
                } while (r.rows == 0);
            }
        }
        if (done()) return false;
        set(a, per);
        return true;
    }
};

// A ring's next slot and the parity of its use.
template <int kSlots> struct Ring {
    int slot = 0, phase = 0;
    __device__ __forceinline__ void step() {
        if (++slot == kSlots) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// kFull: D = 64 kPanels, every step of the first product.  kShaped: capped
// scores, a decay or a scale that is not positive.
template <typename T, int kPanels, bool kFull, bool kShaped>
__global__ void __launch_bounds__(kThreads, 1)
attn_chunk_kernel(const AttnArgs a, const AttnWork w, const ChunkStart* starts, const __grid_constant__ CUtensorMap map_q,
                  const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using L = Layout<kPanels>;
    extern __shared__ uint8_t s_raw[];
    uint8_t* s_q = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* s_kv = s_q + L::kQ;
    __shared__ uint64_t s_qfull, s_qempty, s_full[L::kSlots], s_ready[L::kSlots], s_empty[L::kSlots];
    __shared__ uint64_t s_sfull[2][2], s_pfull[2][2], s_odone[2][2], s_drain[2];      // [row tile][half]
    __shared__ uint32_t s_tmem;
    __shared__ int s_err;
    const WaitLimit limit{&s_err, w.wait_ns};
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per = kRows / a.group;              // tokens of a row tile
    const int ksteps = (a.D + 15) / 16;

    if (tid == 0) {
        s_err = 0;
        mbar_init(&s_qfull, 1);
        mbar_init(&s_qempty, 2);
        for (int i = 0; i < L::kSlots; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_ready[i], 1);
            mbar_init(&s_empty[i], 2);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_sfull[i >> 1][i & 1], 1);
            mbar_init(&s_pfull[i >> 1][i & 1], 4);
            mbar_init(&s_odone[i >> 1][i & 1], 1);
        }
        mbar_init(&s_drain[0], 1);
        mbar_init(&s_drain[1], 1);
        fence_mbar_init();
        prefetch_tmap(&map_q);
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
    }
    if (warp == 1) {
        tmem_alloc(&s_tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    launch_dependents();
    wait_primary();                               // the shares

    bool ok = true;
    if (warp < 4) {
        Walk k;
        bool more = k.start(a, starts, blockIdx.x, per);
        if (warp == 0) {
            // ---- loads -------------------------------------------------------------
            const int boxes = kTile / w.box;
            const bool on = lane < boxes * kPanels;
            const int panel = lane / boxes, at = (lane % boxes) * w.box;
            int slot_no = 0, q_no = 0;
            if (blockIdx.x == w.stall) more = false;
            for (; more && ok; more = k.next(a, per)) {
                if (k.begin == k.end) continue;       // nothing visible: no tile, no query
                if (q_no > 0 && !warp_wait<true>(&s_qempty, (q_no - 1) & 1, limit, 1)) { ok = false; break; }
                ++q_no;
                if (lane == 0) mbar_arrive_expect_tx(&s_qfull, k.u.nq * kPanels * per * a.group * 128);
                __syncwarp();
                if (lane < k.u.nq * kPanels)
                    tma_load_4d(s_q + lane * L::kPanel, &map_q, &s_qfull, (lane % kPanels) * 64, 0, k.cur.h,
                                k.r.first + k.u.row0 + (lane / kPanels) * per);
                const int32_t* table = a.tables + (int64_t)k.cur.b * a.pitch;
                auto entry_of = [&](int t) {          // the table's, of this lane's box; -1: none
                    const int key = key_of(k.u, t) + at;
                    return on && key < k.r.len ? table[key / a.page] : -1;
                };
                int entry = entry_of(k.begin);
                for (int t = k.begin; t < k.end && ok; ++t) {
                    // num_pages reads as 0
                    const int off = (key_of(k.u, t) + at) % a.page;
                    const int page = entry >= 0 && entry < a.num_pages ? entry : a.num_pages;
                    if (t + 1 < k.end) entry = entry_of(t + 1);       // used a tile later: its latency is hidden
#pragma unroll
                    for (int side = 0; side < 2; ++side, ++slot_no) {
                        const int slot = slot_no % L::kSlots, phase = (slot_no / L::kSlots) & 1;
                        if (slot_no >= L::kSlots && !warp_wait<true>(&s_empty[slot], phase ^ 1, limit, 2)) {
                            ok = false;
                            break;
                        }
                        if (lane == 0) mbar_arrive_expect_tx(&s_full[slot], L::kSlot);
                        __syncwarp();
                        if (on)
                            tma_load_4d(s_kv + slot * L::kSlot + panel * L::kPanel + at * 128, side == 0 ? &map_k : &map_v,
                                        &s_full[slot], panel * 64, off, k.cur.h, page);
                    }
                }
            }
            // no copy may be in flight when the CTA ends
            for (int i = max(0, slot_no - L::kSlots); i < slot_no; ++i)
                drain_wait<true>(&s_full[i % L::kSlots], (i / L::kSlots) & 1, limit, 3);
            if (q_no > 0) drain_wait<true>(&s_qfull, (q_no - 1) & 1, limit, 3);
        } else if (warp != 2) {
            // ---- products of row tile t ----------------------------------------------
            // The warp stays together: every lane walks and waits, an elected one issues.
            // The operands of tcgen05.mma are uniform registers; in code that a single
            // lane runs by a comparison (lane == 0) they would be copies of that lane's.
            const int t = warp == 1 ? 0 : 1;
            const uint32_t bf = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            const uint32_t idesc_s = idesc_f16(kRows, kHalf) | bf;
            const uint32_t idesc_o = idesc_f16(kRows, ksteps * 16) | bf | (1u << 16);      // B: columns contiguous
            // What leads up to an instruction has to be short: of a descriptor only the low
            // word changes, by an add on its address field (16-byte units).
            const uint32_t q_lo = ((smem_u32(s_q) >> 4) | (1u << 16)) + (uint32_t)(t * (kPanels * L::kPanel / 16));
            const uint32_t k_lo = (smem_u32(s_kv) >> 4) | (1u << 16);
            const uint32_t v_lo = (smem_u32(s_kv) >> 4) | ((uint32_t)L::kPanel >> 4) << 16;
            const uint32_t tm_s = tmem + t * 128, tm_o = tmem + 256 + t * 128;
            Ring<L::kSlots> keys, vals, vready;       // the ring's slots of keys and values (every other one), value tiles
            vals.step();
            int q_no = 0, steps[2] = {0, 0};          // queries freed; weights multiplied, by half
            int s_done = 0;                           // scores made of second halves
            auto wait = [&](uint64_t* bar, int phase, int code) {
                ok = ok && warp_wait<true>(bar, phase & 1, limit, code);
                return ok;
            };
            // S = Q K^T of 64 keys.  It overwrites P: products with different accumulators
            // are not ordered by their issue, so the one that reads P has to be done.
            auto scores = [&](int h, int slot) {
                tc_fence_after();
                const uint32_t kb = k_lo + (uint32_t)(slot * (L::kSlot / 16) + h * (kHalf * 128 / 16));
                if (kFull) {
                    mma_scores<kPanels>(tm_s + h * kHalf, q_lo, kb, idesc_s, &s_sfull[t][h]);
                } else {
                    for (int ks = 0; ks < ksteps; ++ks) {
                        const uint32_t off = (uint32_t)((ks >> 2) * (L::kPanel / 16) + (ks & 3) * 2);
                        if (elect_one()) mma_f16_lo(tm_s + h * kHalf, q_lo + off, kb + off, idesc_s, ks > 0 ? 1u : 0u);
                    }
                    if (elect_one()) mma_commit(&s_sfull[t][h]);
                }
                s_done += h;
            };
            // O (+)= P V of 64 keys, once the weights are there.
            auto outputs = [&](int h, bool add) {
                if (!wait(&s_pfull[t][h], steps[h], 9)) return false;
                tc_fence_after();
                mma_weights(tm_o, tm_s + h * kHalf, v_lo + (uint32_t)(vals.slot * (L::kSlot / 16) + h * (kHalf * 128 / 16)), idesc_o,
                            add, &s_odone[t][h]);
                ++steps[h];
                return true;
            };
            auto outputs_done = [&](int h) { return steps[h] == 0 || wait(&s_odone[t][h], steps[h] - 1, 13); };
            auto values_there = [&] { return wait(&s_full[vals.slot], vals.phase, 6) && wait(&s_ready[vready.slot], vready.phase, 7); };
            auto two_on = [](Ring<L::kSlots>& r) { r.step(); r.step(); };
            // What frees a slot is known here without a commit of its own (which would wait
            // in the queue behind the products): weights follow from finished scores, and
            // S waits for finished outputs.
            auto free = [&](uint64_t* bar) {
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            for (; more && ok; more = k.next(a, per)) {
                const int n = __shfl_sync(0xffffffffu, k.end - k.begin, 0);
                const int mine = __shfl_sync(0xffffffffu, t == 0 ? k.count[0] : k.count[1], 0);
                if (n == 0) continue;
                if (!wait(&s_qfull, q_no, 4) || !wait(&s_full[keys.slot], keys.phase, 5)) break;
                if (mine > 0) {
                    if (!outputs_done(0) || !outputs_done(1)) break;
                    scores(0, keys.slot);
                    scores(1, keys.slot);
                    if (!values_there()) break;
                }
#pragma unroll 1
                for (int j = 0; j < mine && ok; ++j) {
                    // here: scores of tile j made, its values there.  The waits for what comes by
                    // TMA stand where the products' own take time.
                    const bool next = j + 1 < mine;
                    uint64_t* this_keys = &s_empty[keys.slot];
                    uint64_t* this_vals = &s_empty[vals.slot];
                    two_on(keys);
                    if (!outputs(0, j > 0)) break;
                    if (j + 1 < n && !wait(&s_full[keys.slot], keys.phase, 8)) break;
                    if (next) {
                        if (!outputs_done(0)) break;
                        scores(0, keys.slot);
                    }
                    if (!outputs(1, true)) break;
                    free(this_keys);
                    if (j + 1 == n) free(&s_qempty);
                    two_on(vals);
                    vready.step();
                    if (next && !values_there()) break;
                    if (!outputs_done(1)) break;
                    free(this_vals);
                    if (next) scores(1, keys.slot);
                }
                if (!ok) break;
                // tiles that only the other row tile sees
#pragma unroll 1
                for (int j = mine; j < n; ++j) {
                    if (!wait(&s_full[keys.slot], keys.phase, 5) || !values_there()) break;
                    free(&s_empty[keys.slot]);
                    free(&s_empty[vals.slot]);
                    if (j + 1 == n) free(&s_qempty);
                    two_on(keys);
                    two_on(vals);
                    vready.step();
                }
                ++q_no;
            }
            // No product may be in flight when TMEM is freed, and no commit's arrival
            // when the CTA's shared memory is: the last of each barrier is awaited.
            if (elect_one()) mma_commit(&s_drain[t]);
            drain_wait<true>(&s_drain[t], 0, limit, 10);
            if (steps[0] > 0) drain_wait<true>(&s_odone[t][0], (steps[0] - 1) & 1, limit, 10);
            if (steps[1] > 0) drain_wait<true>(&s_odone[t][1], (steps[1] - 1) & 1, limit, 10);
            if (s_done > 0) drain_wait<true>(&s_sfull[t][1], (s_done - 1) & 1, limit, 10);
            __syncwarp();
        } else {
            // ---- values that no row sees ----------------------------------------------
            Ring<L::kSlots> ring, vring;
            for (; more && ok; more = k.next(a, per)) {
                for (int t = k.begin; t < k.end; ++t) {
                    // The keys too, in the ring's order: loads land in any order, and a
                    // parity tells only neighbouring uses of a slot apart.
                    ok = ok && warp_wait<true>(&s_full[ring.slot], ring.phase, limit, 10);
                    if (!ok) break;
                    ring.step();
                    const int slot = ring.slot;
                    ok = ok && warp_wait<true>(&s_full[slot], ring.phase, limit, 10);
                    if (!ok) break;
                    ring.step();
                    const int key0 = key_of(k.u, t);
                    if (!(key0 + kTile <= k.r.prefix || (key0 >= k.u.low && key0 + kTile <= k.u.high))) {
                        const uint32_t v = smem_u32(s_kv) + slot * L::kSlot;
                        for (int i = lane; i < kTile; i += 32) {
                            const int j = key0 + i;
                            if (!(j < k.r.prefix || (j >= k.u.low && j < k.u.high)))
                                for (int c = 0; c < kPanels * 8; ++c)
                                    st_shared_zero16(v + (c >> 3) * L::kPanel + i * 128 + (c & 7) * 16);
                        }
                        fence_proxy_async();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_ready[vring.slot]);      // by value tile: a slot may hold keys next
                    vring.step();
                }
            }
        }
    } else {
        // ---- softmax: warpgroup t, a thread for each row ------------------------------
        Walk k;
        bool more = k.start(a, starts, blockIdx.x, per);
        const int t = (warp - 4) >> 2, row = tid - 128 - t * 128;
        const uint32_t tm_s = tmem + ((uint32_t)(warp & 3) << 21) + t * 128;      // lanes of this warp
        const uint32_t tm_o = tm_s + 256;
        int seen_tiles = 0;                       // the phase of each half's barriers
        for (; more && ok; more = k.next(a, per)) {
            if (t >= k.u.nq) continue;
            const int n = t == 0 ? k.count[0] : k.count[1];
            const int tok0 = k.u.row0 + t * per, toks = min(per, k.u.rows - t * per);
            const int tok = tok0 + row / a.group, head = k.cur.h * a.group + row % a.group;
            const bool valid = row < toks * a.group;
            const int pos = k.r.len - k.r.rows + tok;
            const int hi = valid ? min(k.r.len, pos + 1) : 0, pre = valid ? k.r.prefix : 0;
            const int lo = a.window > 0 ? pos - a.window + 1 : 0;
            const float decay = valid && a.decay != nullptr ? a.decay[head] * kLog2e : 0.0f;
            // keys that all rows of the tile see, besides the prefix
            const int first_pos = k.r.len - k.r.rows + tok0;
            const int all_hi = min(k.r.len, first_pos + 1), all_lo = a.window > 0 ? first_pos + toks - a.window : 0;
            // A lane without a row has scores of whatever lies there (another request's queries,
            // an earlier launch's shared memory).  Its maximum is out of reach from the start, so
            // that it never moves those of the warp's rows.
            float m = valid ? -INFINITY : INFINITY, l = 0.0f;

            for (int j = 0; j < n && ok; ++j) {
                const int key_tile = key_of(k.u, k.begin + j);
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    ok = ok && warp_wait<true>(&s_sfull[t][h], seen_tiles & 1, limit, 11);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t tm = tm_s + h * kHalf;
                    uint32_t sr[kHalf];               // the row's scores
                    tmem_load(tm, sr);
                    const int key0 = key_tile + h * kHalf;
                    const bool all = key0 + kHalf <= k.r.prefix || (key0 >= all_lo && key0 + kHalf <= all_hi);
                    float f = a.scale * kLog2e, top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (kShaped) {
                        // the score in units of log 2 itself
                        if (a.softcap > 0.0f) {
                            float far = 0.0f;         // the largest |score| of the row
#pragma unroll
                            for (int i = 0; i < kHalf; i += 2)
                                far = max3(far, fabsf(__uint_as_float(sr[i])), fabsf(__uint_as_float(sr[i + 1])));
                            // The score alone says which form of tanh it takes; the vote
                            // says only whether the warp needs the second one.
                            if (__all_sync(0xffffffffu, (hi | pre) == 0 || cap_is_small(far, a.cap))) {
#pragma unroll
                                for (int i = 0; i < kHalf; i += 2) {
                                    const float2 e = cap_small(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1]), a.cap);
                                    sr[i] = __float_as_uint(e.x);
                                    sr[i + 1] = __float_as_uint(e.y);
                                }
                            } else {
                                // In place in TMEM, 16 columns at a time: written out over all 64 in
                                // registers, this way took 281 us for 8 capped chunks instead of 216 and
                                // the one above 187 instead of 178 (32 at a time: 228 and 185).
#pragma unroll 1
                                for (int c = 0; c < 4; ++c) {
                                    uint32_t x[16];
                                    tmem_load(tm + c * 16, x);
#pragma unroll
                                    for (int i = 0; i < 16; i += 2) {
                                        const float2 e = cap_any(__uint_as_float(x[i]), __uint_as_float(x[i + 1]), a.cap);
                                        x[i] = __float_as_uint(e.x);
                                        x[i + 1] = __float_as_uint(e.y);
                                    }
                                    tmem_st_32x32b_x16(tm + c * 16, x);
                                }
                                tmem_st_wait();
                                tmem_load(tm, sr);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < kHalf; ++i) sr[i] = __float_as_uint(__uint_as_float(sr[i]) * f);
                        }
                        if (a.decay != nullptr) {
                            const float age = (float)(pos - key0);
                            const uint64_t rate = pair(-decay, -decay), age2 = pair(age, age);
                            if (key0 + kHalf <= first_pos + 1) {      // no key ahead of a row
#pragma unroll
                                for (int i = 0; i < kHalf; i += 2) {
                                    const float2 e = split(fma2(rate, add2(age2, pair(-(float)i, -(float)(i + 1))),
                                                                pair(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1]))));
                                    sr[i] = __float_as_uint(e.x);
                                    sr[i + 1] = __float_as_uint(e.y);
                                }
                            } else {
#pragma unroll
                                for (int i = 0; i < kHalf; ++i)
                                    sr[i] = __float_as_uint(fmaf(-decay, fmaxf(age - (float)i, 0.0f), __uint_as_float(sr[i])));
                            }
                        }
                        f = 1.0f;
                    }
                    if (!all) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int kb = key0 + c * 32;
                            const uint32_t seen = low_bits(pre - kb) | (low_bits(hi - kb) & ~low_bits(lo - kb));
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!((seen >> i) & 1u)) sr[c * 32 + i] = 0xff800000u;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kHalf; i += 2)
                        top4[(i >> 1) & 3] = max3(top4[(i >> 1) & 3], __uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
                    const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * f;      // f > 0
                    if (__any_sync(0xffffffffu, top > m + kSlack)) {      // m = -inf at first
                        const float to = fmaxf(top, m);
                        const float keep = to == -INFINITY ? 1.0f : exp2f_fast(m - to);
                        if (j + h > 0) {
                            // once the products of the steps before are in O
                            ok = ok && warp_wait<true>(&s_odone[t][h ^ 1], (seen_tiles + h + 1) & 1, limit, 14);
                            if (!ok) break;
                            tc_fence_after();
                            for (int c = 0; c * 32 < a.D; ++c) {
                                uint32_t o[32];
                                tmem_load(tm_o + c * 32, o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                                tmem_st_32x32b_x32(tm_o + c * 32, o);
                            }
                        }
                        l *= keep;
                        m = to;
                    }
                    const float base = m == -INFINITY ? 0.0f : m;
                    const uint64_t f2 = pair(f, f), base2 = pair(-base, -base);
                    uint64_t sum[4] = {0, 0, 0, 0};
                    uint32_t p[kHalf / 2];
#pragma unroll
                    for (int i = 0; i < kHalf / 2; ++i) {
                        const float2 e = split(fma2(pair(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), f2, base2));
                        const float x = exp2f_fast(e.x), y = exp2f_fast(e.y);
                        sum[i & 3] = add2(sum[i & 3], pair(x, y));
                        p[i] = pack2<T>(x, y);
                    }
                    tmem_st_32x32b_x32(tm, p);
                    {
                        const float2 e = split(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
                        l += e.x + e.y;
                    }
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_pfull[t][h]);
                }
                ++seen_tiles;
            }
            if (!ok) break;

            // ---- the piece's end -------------------------------------------------
            // the product of the last step, which those before it are part of
            if (n > 0) {
                ok = ok && warp_wait<true>(&s_odone[t][1], (seen_tiles - 1) & 1, limit, 12);
                if (!ok) break;
                tc_fence_after();
            }
            const bool whole = k.begin == 0 && k.end == k.u.tiles;
            const int slot = 2 * blockIdx.x + (k.begin == 0);
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T* out = reinterpret_cast<T*>(a.out) + (int64_t)(k.r.first + tok) * a.o_tok + (int64_t)head * a.o_head;
            float* part = w.chunk_o + (int64_t)slot * kPartCols * 2 * kRows + t * kRows + row;
            // TMEM loads are for the whole warp: lanes without a row take part, and all
            // are together again before the next one.
#pragma unroll
            for (int c = 0; c < 2 * kPanels; ++c) {
                if (c * 32 < a.D) {
                    uint32_t o[32];
                    __syncwarp();
                    if (n > 0) {
                        tmem_load(tm_o + c * 32, o);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0;
                    }
                    if (valid && whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            if (c * 32 + i < a.D) {
                                uint32_t p[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    p[e] = pack2<T>(__uint_as_float(o[i + 2 * e]) * inv, __uint_as_float(o[i + 2 * e + 1]) * inv);
                                *reinterpret_cast<uint4*>(out + c * 32 + i) = make_uint4(p[0], p[1], p[2], p[3]);
                            }
                        }
                    } else if (valid) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (c * 32 + i < a.D) part[(int64_t)(c * 32 + i) * 2 * kRows] = __uint_as_float(o[i]);
                    }
                    __syncwarp();
                }
            }
            if (valid && whole && a.lse != nullptr)
                a.lse[(int64_t)(k.r.first + tok) * a.hq + head] = log_sum(m, l);
            if (valid && !whole) w.chunk_ml[slot * 2 * kRows + t * kRows + row] = make_float2(m, l);
        }
    }
    if (lane == 0) report_wait(limit, w.host_err, w.failed + blockIdx.x);
    tc_fence_before();
    __syncthreads();
    if (*(volatile int*)&s_err != 0)              // this CTA's parts of cut units have no result
        for (int i = tid; i < 4 * kRows; i += kThreads) w.chunk_ml[2 * blockIdx.x * 2 * kRows + i] = make_float2(0.0f, NAN);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- cut units ----------------------------------------------------------------

// Whole units of a CTA whose wait gave up: NaN in each of its rows.
template <typename T>
__device__ void mark_units(const AttnArgs& a, const ChunkStart* starts, int cta) {
    const int per = kRows / a.group, t = threadIdx.x / kRows, row = threadIdx.x % kRows;
    Walk k;
    for (bool more = k.start(a, starts, cta, per); more; more = k.next(a, per)) {
        const int toks = min(per, k.u.rows - t * per);
        if (k.begin != 0 || k.end != k.u.tiles || row >= toks * a.group) continue;
        const int64_t tok = k.r.first + k.u.row0 + t * per + row / a.group;
        const int head = k.cur.h * a.group + row % a.group;
        T* out = reinterpret_cast<T*>(a.out) + tok * a.o_tok + (int64_t)head * a.o_head;
        const uint32_t none = pack2<T>(NAN, NAN);
        for (int d = 0; d < a.D; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(none, none, none, none);
        if (a.lse != nullptr) a.lse[tok * a.hq + head] = NAN;
    }
}

constexpr int kJoinBlocks = 2 * kRows / 32;

// Block (i, group of 32 rows): if share i begins inside a unit and is the first
// to, joins the unit's parts, in their order: share i-1's end, then i, i+1, ...
// Rows that a CTA left without a result, because a wait of it gave up, get NaN:
// in cut units by their parts' sums, in whole ones here, by the blocks of a row
// group more (neither costs the kernels' loops anything).
template <typename T>
__global__ void __launch_bounds__(256) attn_chunk_join_kernel(const AttnArgs a, const AttnWork w, const ChunkStart* starts,
                                                              int ctas) {
    wait_primary();
    const int i = blockIdx.x + 1;
    if (blockIdx.y == kJoinBlocks) {
        if (w.failed[i] != 0) mark_units<T>(a, starts, i);
        if (i == 1 && w.failed[0] != 0) mark_units<T>(a, starts, 0);
        return;
    }
    const ChunkStart s = starts[i], p = starts[i - 1];
    if (s.b >= a.B || s.tile == 0) return;
    if (p.b == s.b && p.qt == s.qt && p.h == s.h && p.tile > 0) return;      // cut before
    int parts = 2;
    while (i + parts - 1 < ctas) {
        const ChunkStart x = starts[i + parts - 1];
        if (x.b != s.b || x.qt != s.qt || x.h != s.h || x.tile == 0) break;
        ++parts;
    }
    const int per = kRows / a.group;
    const Request r = load_request(a, s.b);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.y * 32 + lane, t = row / kRows, in = row - t * kRows;
    const int tok = s.qt * 2 * per + t * per + in / a.group;
    if (in >= per * a.group || tok >= r.rows) return;
    auto slot = [&](int n) { return 2 * (i - 1 + n) + (n == 0); };
    float top = -INFINITY, sum = 0.0f;
    for (int n = 0; n < parts; ++n) top = fmaxf(top, w.chunk_ml[slot(n) * 2 * kRows + row].x);
    for (int n = 0; n < parts; ++n) {
        const float2 ml = w.chunk_ml[slot(n) * 2 * kRows + row];
        sum += scaled_sum(ml.x, ml.y, top);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int head = s.h * a.group + in % a.group;
    T* out = reinterpret_cast<T*>(a.out) + (int64_t)(r.first + tok) * a.o_tok + (int64_t)head * a.o_head;
    for (int d = warp * 8; d < a.D; d += 64) {
        float v[8] = {};
#pragma unroll 2
        for (int n = 0; n < parts; ++n) {
            const float pm = w.chunk_ml[slot(n) * 2 * kRows + row].x;
            const float f = pm == -INFINITY ? 0.0f : exp2f_fast(pm - top);
            const float* o = w.chunk_o + (int64_t)slot(n) * kPartCols * 2 * kRows + row;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += f * o[(int64_t)(d + e) * 2 * kRows];
        }
        *reinterpret_cast<uint4*>(out + d) =
            make_uint4(pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv),
                       pack2<T>(v[4] * inv, v[5] * inv), pack2<T>(v[6] * inv, v[7] * inv));
    }
    if (warp == 0 && a.lse != nullptr)
        a.lse[(int64_t)(r.first + tok) * a.hq + head] = log_sum(top, sum);
}

// Launches a kernel whose set-up may overlap the end of the one before it in the
// stream (programmatic dependent launch; it waits for that one itself).
template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    MARS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
    return MARS_OK;
}

template <typename T, int kPanels, bool kFull, bool kShaped>
int launch(const AttnArgs& a, const AttnWork& w, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
           int ctas, cudaStream_t st) {
    using L = Layout<kPanels>;
    static std::atomic<uint64_t> done{0};
    MARS_TRY(allow_smem(reinterpret_cast<const void*>(attn_chunk_kernel<T, kPanels, kFull, kShaped>), L::kSmem, done));
    attn_chunk_plan_kernel<<<1, kPlanThreads, a.B * sizeof(int), st>>>(a, w.starts, w.failed, ctas);
    MARS_CUDA_TRY(cudaGetLastError());
    MARS_TRY(launch_after(attn_chunk_kernel<T, kPanels, kFull, kShaped>, dim3(ctas), kThreads, L::kSmem, st, a, w,
                          (const ChunkStart*)w.starts, mq, mk, mv));
    if (ctas > 1)
        MARS_TRY(launch_after(attn_chunk_join_kernel<T>, dim3(ctas - 1, kJoinBlocks + 1), 256, 0, st, a, w,
                              (const ChunkStart*)w.starts, ctas));
    return MARS_OK;
}

}  // namespace

namespace mars {

int attn_chunk(const AttnArgs& a, AttnWork w, const mars_kv_cache* cache, int num_sms, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    w.box = page_box(cache->page_size, kTile);
    MARS_TRY(page_maps(cache, w.box, &mk, &mv));
    MARS_TRY(query_map(a, cache->dtype, kRows / a.group, &mq));
    // scores that a positive factor alone turns into exponents, or not
    const bool shaped = a.softcap > 0.0f || a.decay != nullptr || !(a.scale > 0.0f);
    auto go = [&](auto type, auto panels) {
        using T = decltype(type);
        constexpr int kPanels = decltype(panels)::value;
        if (a.D == 64 * kPanels)
            return shaped ? launch<T, kPanels, true, true>(a, w, mq, mk, mv, num_sms, st)
                          : launch<T, kPanels, true, false>(a, w, mq, mk, mv, num_sms, st);
        return shaped ? launch<T, kPanels, false, true>(a, w, mq, mk, mv, num_sms, st)
                      : launch<T, kPanels, false, false>(a, w, mq, mk, mv, num_sms, st);
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    if (cache->dtype == MARS_DTYPE_F16) return a.D <= 64 ? go(__half(), one) : go(__half(), two);
    return a.D <= 64 ? go(__nv_bfloat16(), one) : go(__nv_bfloat16(), two);
}

}  // namespace mars
