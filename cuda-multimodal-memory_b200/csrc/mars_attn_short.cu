// mars_attn_short.cu -- attention over the paged cache for requests with few
// new tokens (decoding, a drafted handful): a tile has 16 rows, the query heads
// of one key head times its new tokens.
//
// Bound: HBM.  Every key and value is read once for 16 rows, 4 D flops a row
// for 4 D bytes, far below the card's balance, so the kernel is a stream of
// TMA loads with as little as possible between them.
//
//  * Split.  The work is the sequence of all (request, row tile, key head)
//    units' tiles of keys; every CTA takes an equal share of that sequence, as
//    many shares as CTAs fit the card.  Any mix of lengths is balanced to one
//    tile, a long cache is split over all SMs and short ones share a CTA.  The
//    shares follow from the lengths alone, which every CTA sums up by itself
//    (no planning launch, nothing on the host).  A unit cut by a share's end
//    leaves (max, sum, accumulators) in the workspace; the CTA that arrives
//    last (a counter per unit, no spinning) joins the parts in their order, so
//    the result does not depend on timing.
//  * Pipeline.  One producer warp, a lane for each box of a page, fills a ring
//    of 96 KB (two CTAs an SM: 192 KB in flight, three times what latency x
//    bandwidth asks for).  Four consumer warps take a quarter of a tile's keys each and
//    keep a running maximum, sum and accumulator of their own, so nothing but
//    the ring's barriers joins them before a unit's end.
//  * mma.sync m16n8k16.  16 rows are one of its tiles; a tcgen05 tile has 128,
//    of which decoding would fill 1 to 16.  The scores' registers are the
//    second product's operand as they stand.  Rate: 512 of the 2,800 cycles
//    that a 128-key tile takes from HBM.
//
// Measured (bf16, D = 128): 64 requests of up to 8,000 keys, 32 heads on 8:
// 201 us (198 to 212 from card to card), 6.28 TB/s, 0.97 of the copy rate; with a
// cap of 30 203 us, scores beyond half of it 206.  2 requests of up to 250,000,
// 16 heads on 4: 134 us, 0.89; there a unit is cut into 74 parts, and its joining
// is what the other has not (it was 156 us with one thread a row to join).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "mars_attn.cuh"
#include "mars_attn_mma.cuh"
#include "mars_kv.h"
#include "mars_sm100.cuh"

using namespace mars;
using namespace mars::sm100;

namespace {

constexpr int kRows = kShortRows;               // 16
constexpr int kConsumers = 4;                   // warps
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr int kRing = 96 * 1024;

// A tile is 32 KB of keys and values: 128 keys of up to 64 columns, 64 of up to
// 128.  (64 keys of 64 columns, 16 KB, left what a tile costs beside its bytes
// -- barriers, masks, maxima, rescaling -- in the way: 4 requests of 700 keys
// 14.4 us, with 128 keys 11.3.)
template <int kPanels> struct Layout {
    static constexpr int kTile = 128 / kPanels;                   // keys
    static constexpr int kPer = kTile / kConsumers;               // of a warp: 32 or 16
    static constexpr int kStage = 2 * kPanels * kTile * 128;      // bytes: keys, then values
    static constexpr int kStages = kRing / kStage;
    static constexpr int kCols = 64 * kPanels;
    static constexpr int kPitch = kCols + 8;                      // floats of a row of s_o: no bank conflicts
    static constexpr int kSmem = 1024 + kRing + kRows * kPitch * 4;
};

// One unit: row tile qt of request b, its key tiles.
struct Unit {
    int row0, rows;               // tokens of the tile
    int n1, s2, tiles;            // tiles of the prefix; first tile of the rest; in all
    int low, high;                // the rest's keys
};

template <int kTile>
__device__ __forceinline__ Unit make_unit(const AttnArgs& a, const Request& r, int qt, int per) {
    Unit u;
    u.row0 = qt * per;
    u.rows = min(per, r.rows - u.row0);
    row_range(a, r, u.row0, u.row0 + u.rows, &u.low, &u.high);
    u.n1 = (r.prefix + kTile - 1) / kTile;
    u.s2 = max(u.n1, u.low / kTile);
    u.tiles = u.n1 + max(0, (u.high + kTile - 1) / kTile - u.s2);
    return u;
}

// Where the sequence of shares stands.
struct Cursor {
    int b, qt, h, tile;
    long long left;               // tiles of the share from here on
};

struct Found { int b, qt, h, tile; };

template <typename T, int kPanels>
__global__ void __launch_bounds__(kThreads, 2) attn_short_kernel(const AttnArgs a, const AttnWork w,
                                                                 const __grid_constant__ CUtensorMap map_k,
                                                                 const __grid_constant__ CUtensorMap map_v) {
    using L = Layout<kPanels>;
    constexpr int kTile = L::kTile, kBlocks = L::kPer / 8;        // blocks of 8 keys a warp
    extern __shared__ uint8_t s_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~(uintptr_t)1023);
    float* s_o = reinterpret_cast<float*>(ring + kRing);
    __shared__ uint64_t s_full[L::kStages], s_empty[L::kStages];
    __shared__ float s_m[kConsumers][kRows], s_l[kConsumers][kRows], s_top[kRows], s_inv[kRows];
    __shared__ long long s_sum[kThreads / 32 + 1];
    __shared__ Found s_found;
    __shared__ int s_last, s_err;
    const WaitLimit limit{&s_err, w.wait_ns};
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per = kRows / a.group;              // tokens of a row tile

    if (tid == 0) {
        s_err = 0;
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], kConsumers);
        }
        fence_mbar_init();
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
    }

    // ---- this CTA's share: [x0, x1) of the sequence of tiles ----------------
    const int each = (a.B + kThreads - 1) / kThreads;
    const int b0 = min(a.B, tid * each), b1 = min(a.B, b0 + each);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
        const Request r = load_request(a, b);
        for (int qt = 0; qt * per < r.rows; ++qt) mine += max(1, make_unit<kTile>(a, r, qt, per).tiles);
    }
    mine *= a.hkv;
    long long upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += o;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    long long before = upto - mine, total = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
        if (i < warp) before += s_sum[i];
        total += s_sum[i];
    }
    const long long share = max((total + gridDim.x - 1) / gridDim.x, (long long)w.min_share);
    const long long x0 = blockIdx.x * share, x1 = min(total, x0 + share);
    if (x0 >= total) return;
    if (before <= x0 && x0 < before + mine) {
        long long x = x0 - before;
        for (int b = b0; b < b1; ++b) {
            const Request r = load_request(a, b);
            for (int qt = 0; qt * per < r.rows; ++qt) {
                const int c = max(1, make_unit<kTile>(a, r, qt, per).tiles);
                if (x >= 0 && x < (long long)c * a.hkv)
                    s_found = Found{b, qt, (int)(x / c), (int)(x % c)};
                x -= (long long)c * a.hkv;
            }
        }
    }
    __syncthreads();

    Cursor cur{s_found.b, s_found.qt, s_found.h, s_found.tile, x1 - x0};
    Request r = load_request(a, cur.b);
    const int T_per_page = a.page;

    if (warp == kConsumers) {
        // ---- producer --------------------------------------------------------
        const int boxes = kTile / w.box;          // of one panel of keys
        const bool on = lane < boxes * kPanels * 2;
        const int panel = (lane / boxes) % kPanels, at = (lane % boxes) * w.box;
        const bool is_v = lane / boxes >= kPanels;
        const CUtensorMap* map = is_v ? &map_v : &map_k;
        const int dst = ((is_v ? kPanels : 0) + panel) * kTile * 128 + at * 128;
        int issued = 0;
        bool ok = blockIdx.x != w.stall;
        while (ok && cur.left > 0) {
            const Unit u = make_unit<kTile>(a, r, cur.qt, per);
            const int c = max(1, u.tiles), end = (int)min((long long)c, cur.tile + cur.left);
            const int32_t* table = a.tables + (int64_t)cur.b * a.pitch;
            auto page_of = [&](int t) {           // of this lane's box in tile t of the unit; num_pages: reads as 0
                const int key = (t < u.n1 ? t : u.s2 + t - u.n1) * kTile + at;
                int page = a.num_pages;
                if (on && key < r.len) {
                    page = table[key / T_per_page];
                    if (page < 0 || page >= a.num_pages) page = a.num_pages;
                }
                return page;
            };
            int page = cur.tile < u.tiles ? page_of(cur.tile) : 0;
            for (int t = cur.tile; t < min(end, u.tiles); ++t) {
                const int stage = issued % L::kStages, phase = (issued / L::kStages) & 1;
                if (issued >= L::kStages &&
                    !warp_wait(&s_empty[stage], phase ^ 1, limit, 1)) { ok = false; break; }
                if (lane == 0) mbar_arrive_expect_tx(&s_full[stage], L::kStage);
                __syncwarp();
                const int key = (t < u.n1 ? t : u.s2 + t - u.n1) * kTile + at;
                if (on)
                    tma_load_4d(ring + stage * L::kStage + dst, map, &s_full[stage], panel * 64, key % T_per_page, cur.h, page);
                ++issued;
                if (t + 1 < end) page = page_of(t + 1);
            }
            cur.left -= end - cur.tile;
            cur.tile = 0;
            if (++cur.h == a.hkv) {
                cur.h = 0;
                if (++cur.qt * per >= r.rows && cur.left > 0) {
                    cur.qt = 0;
                    do r = load_request(a, ++cur.b); while (r.rows == 0);
                }
            }
        }
        // no copy may be in flight when the CTA ends
        for (int i = max(0, issued - L::kStages); i < issued; ++i)
            drain_wait(&s_full[i % L::kStages], (i / L::kStages) & 1, limit, 2);
        if (lane == 0) report_wait(limit, w.host_err);
        return;
    }

    // ---- consumers -----------------------------------------------------------
    const int qr = lane >> 2, qc = (lane & 3) * 2;             // accumulator row (and + 8) and column
    constexpr float kLog2e = 1.4426950408889634f;
    int used = 0;
    bool ok = true;
    while (cur.left > 0) {
        const Unit u = make_unit<kTile>(a, r, cur.qt, per);
        const int c = max(1, u.tiles), begin = cur.tile, end = (int)min((long long)c, begin + cur.left);
        const int head0 = cur.h * a.group, valid = u.rows * a.group;

        // rows qr and qr + 8: token and head, position, the keys they see
        uint32_t qf[4 * kPanels][4];
        int pos[2], lo[2], hi[2], pre[2];
        float decay[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = qr + 8 * i;
            const bool in = row < valid;
            const int tok = u.row0 + row / a.group, head = head0 + row % a.group;
            pos[i] = r.len - r.rows + tok;
            hi[i] = in ? min(r.len, pos[i] + 1) : 0;
            lo[i] = a.window > 0 ? pos[i] - a.window + 1 : 0;
            pre[i] = in ? r.prefix : 0;
            decay[i] = in && a.decay != nullptr ? a.decay[head] * kLog2e : 0.0f;
            const uint32_t* q = reinterpret_cast<const uint32_t*>(
                reinterpret_cast<const T*>(a.q) + (int64_t)(r.first + tok) * a.q_tok + (int64_t)head * a.q_head);
#pragma unroll
            for (int ks = 0; ks < 4 * kPanels; ++ks) {
                qf[ks][i] = in && ks * 16 < a.D ? q[(ks * 16 + qc) / 2] : 0u;
                qf[ks][i + 2] = in && ks * 16 + 8 < a.D ? q[(ks * 16 + 8 + qc) / 2] : 0u;
            }
        }
        // keys that every row sees: [all_lo, all_hi), besides the prefix
        const int first_pos = r.len - r.rows + u.row0;
        const int all_hi = min(r.len, first_pos + 1);
        const int all_lo = a.window > 0 ? first_pos + u.rows - a.window : 0;

        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        float o[8 * kPanels][4];
#pragma unroll
        for (int i = 0; i < 8 * kPanels; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;

        for (int t = begin; t < min(end, u.tiles); ++t, ++used) {
            const int stage = used % L::kStages;
            // a wait that gave up: the unit's barriers are still taken, so that no warp is left at one
            ok = ok && warp_wait(&s_full[stage], (used / L::kStages) & 1, limit, 3);
            if (!ok) continue;
            const int key0 = (t < u.n1 ? t : u.s2 + t - u.n1) * kTile + warp * L::kPer;
            const uint32_t sk = smem_u32(ring + stage * L::kStage) + warp * L::kPer * 128;
            const uint32_t sv = sk + kPanels * kTile * 128;

            // scores of the warp's keys, blocks of 8
            float s[kBlocks][4] = {};
            {
                const int row = lane & 7, tok = ((lane >> 4) << 3) + row, half = (lane >> 3) & 1;
#pragma unroll
                for (int ks = 0; ks < 4 * kPanels; ++ks) {
                    if (ks * 16 < a.D) {
#pragma unroll
                        for (int x = 0; x < kBlocks / 2; ++x) {
                            uint32_t f[4];
                            ldmatrix_x4(f, sk + (ks >> 2) * kTile * 128 + (x * 16 + tok) * 128 +
                                               ((((ks & 3) * 2 + half) ^ row) << 4));
                            mma_16816<T>(s[2 * x], qf[ks], f[0], f[1]);
                            mma_16816<T>(s[2 * x + 1], qf[ks], f[2], f[3]);
                        }
                    }
                }
            }
            // in units of log 2
            if (a.softcap > 0.0f) {
                float far = 0.0f;
#pragma unroll
                for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) far = max3(far, fabsf(s[nb][e]), fabsf(s[nb][e + 1]));
                if (__all_sync(0xffffffffu, cap_is_small(far, a.cap))) {
#pragma unroll
                    for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const float2 v = cap_small(s[nb][e], s[nb][e + 1], a.cap);
                            s[nb][e] = v.x;
                            s[nb][e + 1] = v.y;
                        }
                } else {
#pragma unroll
                    for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const float2 v = cap_any(s[nb][e], s[nb][e + 1], a.cap);
                            s[nb][e] = v.x;
                            s[nb][e + 1] = v.y;
                        }
                }
            } else {
                const float f = a.scale * kLog2e;
#pragma unroll
                for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nb][e] *= f;
            }
            if (a.decay != nullptr) {
#pragma unroll
                for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[nb][e] -= decay[e >> 1] * (float)max(0, pos[e >> 1] - (key0 + nb * 8 + qc + (e & 1)));
            }
            const bool all = key0 + L::kPer <= r.prefix || (key0 >= all_lo && key0 + L::kPer <= all_hi);
            if (!all) {
#pragma unroll
                for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = key0 + nb * 8 + qc + (e & 1), i = e >> 1;
                        if (!(j < pre[i] || (j >= lo[i] && j < hi[i]))) s[nb][e] = -INFINITY;
                    }
                // Values of keys that no row sees may be anything, and 0 x NaN is
                // NaN: put zeros there (a lane half a row of one panel's 128 B).
#pragma unroll
                for (int half = lane; half < 2 * L::kPer; half += 32) {
                    const int j = key0 + (half >> 1);
                    if (!(j < r.prefix || (j >= u.low && j < u.high))) {
#pragma unroll
                        for (int p = 0; p < kPanels; ++p)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                st_shared_zero16(sv + p * kTile * 128 + (half >> 1) * 128 + (half & 1) * 64 + i * 16);
                    }
                }
                fence_proxy_async();               // before the ring's next TMA write of this stage
                __syncwarp();
            }

            float keep[2];
            bool moved = false;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = fmaxf(s[0][2 * i], s[0][2 * i + 1]);
#pragma unroll
                for (int nb = 1; nb < kBlocks; ++nb) x = max3(x, s[nb][2 * i], s[nb][2 * i + 1]);
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                x = fmaxf(x, m[i]);
                moved |= x > m[i];
                keep[i] = x > m[i] ? exp2f_fast(m[i] - x) : 1.0f;      // m = -inf: 0
                m[i] = x;
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int i = 0; i < 8 * kPanels; ++i) {
                    o[i][0] *= keep[0];
                    o[i][1] *= keep[0];
                    o[i][2] *= keep[1];
                    o[i][3] *= keep[1];
                }
                l[0] *= keep[0];
                l[1] *= keep[1];
            }
            const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
            for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[nb][e] = exp2f_fast(s[nb][e] - base[e >> 1]);
                    l[e >> 1] += s[nb][e];
                }
#pragma unroll
            for (int x = 0; x < kBlocks / 2; ++x) {
                const float(&s0)[4] = s[2 * x], (&s1)[4] = s[2 * x + 1];
                const uint32_t pf[4] = {pack2<T>(s0[0], s0[1]), pack2<T>(s0[2], s0[3]), pack2<T>(s1[0], s1[1]),
                                        pack2<T>(s1[2], s1[3])};
                const int row = lane & 7, tok = x * 16 + (((lane >> 3) & 1) << 3) + row, half = lane >> 4;
#pragma unroll
                for (int db = 0; db < 4 * kPanels; ++db) {
                    if (db * 16 < a.D) {
                        uint32_t f[4];
                        ldmatrix_x4_trans(f, sv + (db >> 2) * kTile * 128 + tok * 128 + ((((db & 3) * 2 + half) ^ row) << 4));
                        mma_16816<T>(o[2 * db], pf, f[0], f[1]);
                        mma_16816<T>(o[2 * db + 1], pf, f[2], f[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_empty[stage]);
        }

        // ---- the unit's part of this share: join the four warps ---------------
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if ((lane & 3) == 0) {
                s_m[warp][qr + 8 * i] = m[i];
                s_l[warp][qr + 8 * i] = l[i];
            }
        }
        bar_sync(1, 32 * kConsumers);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) top = fmaxf(top, s_m[x][qr + 8 * i]);
            const float f = m[i] == -INFINITY ? 0.0f : exp2f_fast(m[i] - top);
#pragma unroll
            for (int j = 0; j < 8 * kPanels; ++j) {
                o[j][2 * i] *= f;
                o[j][2 * i + 1] *= f;
            }
        }
        for (int x = 0; x < kConsumers; ++x) {     // in the warps' order: the same sum every time
            if (warp == x) {
#pragma unroll
                for (int j = 0; j < 8 * kPanels; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float2* p = reinterpret_cast<float2*>(s_o + (qr + 8 * i) * L::kPitch + j * 8 + qc);
                        float2 v = make_float2(o[j][2 * i], o[j][2 * i + 1]);
                        if (x > 0) { v.x += p->x; v.y += p->y; }
                        *p = v;
                    }
            }
            bar_sync(1, 32 * kConsumers);
        }
        // 8 threads a row, 16 rows
        const int row = tid >> 3, col0 = tid & 7;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int x = 0; x < kConsumers; ++x) top = fmaxf(top, s_m[x][row]);
#pragma unroll
        for (int x = 0; x < kConsumers; ++x)
            sum += scaled_sum(s_m[x][row], s_l[x][row], top);
        if (*(volatile int*)&s_err != 0) sum = NAN;             // a wait gave up: the rows say so

        const long long at = x1 - cur.left - begin;           // the unit's place in the sequence
        const int c0 = (int)(at / share), parts = (int)((at + c - 1) / share) - c0 + 1;
        bool write = true;
        if (parts > 1) {
            const int slot = 2 * blockIdx.x + (begin == 0);
            float* po = w.part_o + (int64_t)slot * kRows * kPartCols;
            if (row < valid) {
                for (int d = col0 * 4; d < a.D; d += 32)
                    *reinterpret_cast<float4*>(po + row * kPartCols + d) =
                        *reinterpret_cast<const float4*>(s_o + row * L::kPitch + d);
                if (col0 == 0) w.part_ml[slot * kRows + row] = make_float2(top, sum);
            }
            __threadfence();
            bar_sync(1, 32 * kConsumers);
            if (tid == 0) {
                s_last = atomicAdd(w.tickets + c0, 1u) == (unsigned)(parts - 1);
                if (s_last) w.tickets[c0] = 0;
                __threadfence();
            }
            bar_sync(1, 32 * kConsumers);
            write = s_last != 0;
            if (write) {
                // A row's eight threads take every eighth part: a cache split over all SMs
                // has a hundred, and one after another they cost more than its reading.
                const int r_ = min(row, valid - 1);
                top = -INFINITY;
#pragma unroll 4
                for (int p = col0; p < parts; p += 8)
                    top = fmaxf(top, __ldcg(&w.part_ml[(2 * (c0 + p) + (p == 0)) * kRows + r_]).x);
#pragma unroll
                for (int off = 1; off < 8; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                sum = 0.0f;
#pragma unroll 4
                for (int p = col0; p < parts; p += 8) {
                    const float2 ml = __ldcg(&w.part_ml[(2 * (c0 + p) + (p == 0)) * kRows + r_]);
                    sum += scaled_sum(ml.x, ml.y, top);
                }
#pragma unroll
                for (int off = 1; off < 8; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            }
        }
        if (write) {
            if (col0 == 0) {
                s_top[row] = top;
                s_inv[row] = sum == 0.0f ? 0.0f : 1.0f / sum;
                if (row < valid && a.lse != nullptr) {
                    const int tok = r.first + u.row0 + row / a.group, head = head0 + row % a.group;
                    a.lse[(int64_t)tok * a.hq + head] = log_sum(top, sum);
                }
            }
            bar_sync(1, 32 * kConsumers);
            // four columns of a row a thread
            const int chunks = a.D / 4;
            for (int i = tid; i < valid * chunks; i += 32 * kConsumers) {
                const int orow = i / chunks, d = (i - orow * chunks) * 4;
                float4 v;
                if (parts > 1) {
                    v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    const float t0 = s_top[orow];
#pragma unroll 8
                    for (int p = 0; p < parts; ++p) {       // in their order: the same sum every time
                        const int at_row = (2 * (c0 + p) + (p == 0)) * kRows + orow;
                        const float pm = __ldcg(&w.part_ml[at_row]).x;
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(w.part_o + (int64_t)at_row * kPartCols + d));
                        const float f = pm == -INFINITY ? 0.0f : exp2f_fast(pm - t0);
                        v.x += f * y.x;
                        v.y += f * y.y;
                        v.z += f * y.z;
                        v.w += f * y.w;
                    }
                } else {
                    v = *reinterpret_cast<const float4*>(s_o + orow * L::kPitch + d);
                }
                const float inv = s_inv[orow];
                const int tok = r.first + u.row0 + orow / a.group, head = head0 + orow % a.group;
                *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (int64_t)tok * a.o_tok + (int64_t)head * a.o_head + d) =
                    make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
            }
        }
        bar_sync(1, 32 * kConsumers);              // s_o, s_m, s_l are the next unit's

        cur.left -= end - begin;
        cur.tile = 0;
        if (++cur.h == a.hkv) {
            cur.h = 0;
            if (++cur.qt * per >= r.rows && cur.left > 0) {
                cur.qt = 0;
                do r = load_request(a, ++cur.b); while (r.rows == 0);
            }
        }
    }
    if (lane == 0) report_wait(limit, w.host_err);
}

template <typename T, int kPanels>
int launch(const AttnArgs& a, const AttnWork& w, const CUtensorMap& mk, const CUtensorMap& mv, int num_sms, cudaStream_t st) {
    using L = Layout<kPanels>;
    static std::atomic<uint64_t> done{0};
    MARS_TRY(allow_smem(reinterpret_cast<const void*>(attn_short_kernel<T, kPanels>), L::kSmem, done));
    attn_short_kernel<T, kPanels><<<2 * num_sms, kThreads, L::kSmem, st>>>(a, w, mk, mv);
    MARS_CUDA_TRY(cudaGetLastError());
    return MARS_OK;
}

}  // namespace

namespace mars {

int attn_short(const AttnArgs& a, AttnWork w, const mars_kv_cache* cache, int num_sms, cudaStream_t st) {
    CUtensorMap mk, mv;
    w.box = page_box(cache->page_size, a.D <= 64 ? Layout<1>::kTile : Layout<2>::kTile);
    MARS_TRY(page_maps(cache, w.box, &mk, &mv));
    // Small calls: 128 keys a CTA.  A piece costs 2 to 3 us beside its tiles (its rows'
    // queries, the warps' joining, the output), so fewer and larger shares are slower
    // (1 request of 100 keys, 12 heads, in tiles of 64: 7.4 us with 2, 11.0 with 4, 25.5
    // with 12).
    w.min_share = a.D <= 64 ? 1 : 2;
    if (cache->dtype == MARS_DTYPE_F16)
        return a.D <= 64 ? launch<__half, 1>(a, w, mk, mv, num_sms, st) : launch<__half, 2>(a, w, mk, mv, num_sms, st);
    return a.D <= 64 ? launch<__nv_bfloat16, 1>(a, w, mk, mv, num_sms, st)
                     : launch<__nv_bfloat16, 2>(a, w, mk, mv, num_sms, st);
}

}  // namespace mars
