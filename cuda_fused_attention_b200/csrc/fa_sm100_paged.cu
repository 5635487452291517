// Attention of a step's new tokens over a paged K/V cache (sm_100a).

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "fa_sm100_internal.h"
#include "fa_sm100_paged.cuh"
#include "fa_sm100_ptx.cuh"

namespace fa_sm100 {

__device__ unsigned int g_paged_error_word;

struct PagedParams {
    FaPagedPlan plan;
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    __nv_bfloat16* o;
    long long q_token, q_head, o_token, o_head;
    long long k_page, k_head, k_row, v_page, v_head, v_row;
    int page_shift;
    float scale_log2;
    float* partial;             // parts of items that cross a border between CTAs' ranges
};

// A row keeps its exponent base until a score exceeds it by this much in the exp2 domain.
constexpr float kRebase = 16.0f;


// =============================================================================
// Narrow kernel: requests of at most 16 query rows per K/V head (decode steps)
// =============================================================================
// Each K/V byte is used for at most 16 rows, so the cache's bytes bound it: 512 bytes a key at
// D = 128 against 16 * 4 * 128 operations. The work of all requests and K/V heads is one line of
// 64-key tiles (request, then head, then key), and each of the grid's CTAs (two per SM) takes an
// equal stretch of it, whatever the requests' lengths: a request that crosses a border is merged
// from partial results by combine_narrow_kernel. A CTA's warp 4 streams the tiles by TMA through a
// ring that runs on across requests, page by page (a page that is absent reads as zeros); warps
// 0-3 take 16 keys of every tile each, S = Q K^T and O += P V by warp-level matrix instructions
// with Q, P and O in registers, a running maximum and sum per warp, and meet only at a segment's
// end. P is rounded to bf16 for the product with V (its sum is taken before); everything else
// that is kept is 32-bit.
constexpr int kNarrowWarps = 4;
constexpr int kNarrowThreads = (kNarrowWarps + 1) * 32;
constexpr int kNarrowCtasPerSm = 2;
constexpr int kNarrowMinTiles = 2;       // tiles a CTA takes at least
constexpr unsigned long long kTimeoutNs = 1000000000ull;

template <int D>
struct NarrowCfg {
    static constexpr int kTile = kNarrowKeys * D * 2;               // bytes of a K or V tile
    static constexpr int kStage = 2 * kTile;
    static constexpr int kStages = D == 128 ? 3 : 6;                // 96 KB in flight per CTA
    static constexpr int kQuarter = D / 4;                          // columns merged at a time
    static constexpr int kMergeStride = kQuarter + 8;               // floats; the pad spreads rows over banks
    static constexpr int kMergeOff = kStages * kStage;
    static constexpr int kStatsOff = kMergeOff + kNarrowWarps * kNarrowRows * kMergeStride * 4;
    static constexpr int kBarOff = kStatsOff + 2 * kNarrowWarps * kNarrowRows * 4;
    static constexpr int kAbortOff = kBarOff + 2 * kStages * 8;
    static constexpr int kSmemBytes = kAbortOff + 16 + 1024;        // slack for 1024-byte alignment
    static constexpr int kPartFloats = kNarrowRows * (D + 2);       // O [16][D], maxima [16], sums [16]
};

__device__ __forceinline__ void record_paged_timeout(volatile uint32_t* abort_flag, uint32_t site)
{
    *abort_flag = 1u;
    atomicOr(&g_paged_error_word, 1u | (site << 8));
}

// Bounded wait on an mbarrier phase; false once the CTA gives up.
__device__ __forceinline__ bool wait_paged(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t site)
{
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t begin = global_timer_ns();
    for (uint32_t spin = 1;; ++spin) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spin & 7u) == 0u) {
            if (*abort_flag) return false;
            if (global_timer_ns() - begin > kTimeoutNs) {
                record_paged_timeout(abort_flag, site);
                return false;
            }
        }
    }
}

// On the way out after a give-up: a copy that was issued must land before shared memory goes away.
__device__ __forceinline__ void drain_paged(uint32_t bar, uint32_t parity)
{
    const uint64_t begin = global_timer_ns();
    while (!mbar_try_wait(bar, parity))
        if (global_timer_ns() - begin > kTimeoutNs) return;
}

enum PagedSite : uint32_t { kSiteNarrowFull = 32, kSiteNarrowEmpty = 33 };

// A stretch of one (request, K/V head) inside a CTA's range.
struct NarrowSegment {
    int b, h;
    long long first, last;      // the item's tiles on the line: [first, last)
    int tile, count;            // this stretch: tiles [tile, tile + count) of the item
};

__device__ __forceinline__ NarrowSegment narrow_segment(const FaPagedPlan& plan, const long long* start, long long x,
                                                        long long end)
{
    NarrowSegment s;
    s.b = find_request(start, plan.num_seqs, x / plan.kv_heads);
    const long long tiles = start[s.b + 1] - start[s.b], base = start[s.b] * plan.kv_heads;
    s.h = static_cast<int>((x - base) / tiles);
    s.first = base + s.h * tiles;
    s.last = s.first + tiles;
    s.tile = static_cast<int>(x - s.first);
    s.count = static_cast<int>((s.last < end ? s.last : end) - x);
    return s;
}

// Tiles per CTA when `total` are shared out over `ctas`.
__device__ __forceinline__ long long narrow_share(long long total, int ctas)
{
    const long long even = (total + ctas - 1) / ctas;
    return even > kNarrowMinTiles ? even : kNarrowMinTiles;
}

template <int D>
__global__ void __launch_bounds__(kNarrowThreads, kNarrowCtasPerSm)
paged_narrow_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ PagedParams p)
{
    using C = NarrowCfg<D>;
    const FaPagedPlan& plan = p.plan;
    const long long* start = narrow_starts(plan.schedule, plan.num_seqs);
    const long long total = start[plan.num_seqs] * plan.kv_heads;
    const long long share = narrow_share(total, gridDim.x);
    const long long begin = share * blockIdx.x;
    if (begin >= total) return;
    const long long end = begin + share < total ? begin + share : total;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + C::kAbortOff);
    auto full = [&](int s) -> uint32_t { return base + C::kBarOff + static_cast<uint32_t>(s) * 8u; };
    auto empty = [&](int s) -> uint32_t { return base + C::kBarOff + static_cast<uint32_t>(C::kStages + s) * 8u; };
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), kNarrowWarps);
        }
        *abort_flag = 0u;
        fence_mbarrier_init();
    }
    __syncthreads();

    if (warp == kNarrowWarps) {
        // ======================= TMA producer ==================================
        // A tile is boxes of 64 columns by min(page, 64) rows: lane = (page of the tile, K or V, column block).
        constexpr int kBlocks = D / 64;
        const int rows = plan.page_size < kNarrowKeys ? plan.page_size : kNarrowKeys;
        const int pages = kNarrowKeys / rows;
        const bool active = lane < pages * 2 * kBlocks;
        const int page_of_tile = lane / (2 * kBlocks);
        const int is_v = (lane / kBlocks) & 1, block = lane % kBlocks;
        const uint32_t offset = static_cast<uint32_t>(is_v * C::kTile + block * kNarrowKeys * 128 + page_of_tile * rows * 128);
        const void* map = is_v ? static_cast<const void*>(&tm_v) : static_cast<const void*>(&tm_k);
        int it = 0;
        bool ok = true;
        for (long long x = begin; x < end && ok;) {
            const NarrowSegment s = narrow_segment(plan, start, x, end);
            x += s.count;
            const int* table = plan.block_table + static_cast<long long>(s.b) * plan.table_stride;
            const int held = (plan.kv_lens[s.b] + plan.page_size - 1) >> p.page_shift;
            auto page_at = [&](int tile) -> int {
                // num_pages is out of the map's range: such a box reads as zeros.
                const int i = ((tile * kNarrowKeys) >> p.page_shift) + page_of_tile;
                if (!active || i >= held) return plan.num_pages;
                const int page = __ldg(table + i);
                if (page >= 0 && page < plan.num_pages) return page;
                atomicOr(&g_paged_error_word, FA_ERROR_BAD_PAGE);
                return plan.num_pages;
            };
            int page = page_at(s.tile);
            for (int i = 0; i < s.count; ++i, ++it) {
                const int slot = it % C::kStages, use = it / C::kStages;
                const int row = ((s.tile + i) * kNarrowKeys) & (plan.page_size - 1);
                if (use > 0 && !__all_sync(0xffffffffu, wait_paged(empty(slot), (use - 1) & 1, abort_flag, kSiteNarrowEmpty))) {
                    ok = false;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(full(slot), C::kStage);
                __syncwarp();
                if (active)
                    tma_load_4d(base + slot * C::kStage + offset, map, full(slot), block * 64, pages > 1 ? 0 : row, s.h, page);
                if (i + 1 < s.count) page = page_at(s.tile + i + 1);
            }
        }
        if (!ok && lane == 0)
            for (int i = it > C::kStages ? it - C::kStages : 0; i < it; ++i) drain_paged(full(i % C::kStages), (i / C::kStages) & 1);
        return;
    }

    // ======================= consumers =========================================
    constexpr int kSteps = D / 16;
    constexpr int kNTiles = D / 8;
    float* merge = reinterpret_cast<float*>(smem + C::kMergeOff);
    float* stats = reinterpret_cast<float*>(smem + C::kStatsOff);      // [warp][16] maxima, then [warp][16] sums
    const int g = lane >> 2, t = lane & 3;
    const int group = plan.heads / plan.kv_heads;
    const float sl2 = p.scale_log2;
    // ldmatrix rows of this lane within a tile (16 keys per warp), and their swizzle term.
    const int k_row = warp * 16 + (lane & 7) + ((lane >> 4) & 1) * 8, k_chunk = (lane >> 3) & 1;
    const int v_row = warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, v_chunk = (lane >> 4) & 1;
    auto swizzled = [](int row, int chunk) -> uint32_t {
        return static_cast<uint32_t>((chunk >> 3) * kNarrowKeys * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
    };
    int it = 0;
    bool ok = true;
    for (long long x = begin; x < end;) {
        const NarrowSegment s = narrow_segment(plan, start, x, end);
        x += s.count;
        const int token0 = plan.query_start[s.b], n = plan.query_start[s.b + 1] - token0, kv = plan.kv_lens[s.b];
        const int rows = n * group;
        const int head0 = s.h * group;
        // Rows g and g + 8 of the fragments; a row that does not exist is zero and goes nowhere.
        const int tok_a = g / group, tok_b = (g + 8) / group;
        const int limit_a = plan.causal ? kv - n + tok_a : kv - 1, limit_b = plan.causal ? kv - n + tok_b : kv - 1;
        const int first_limit = plan.causal ? kv - n : kv - 1;
        const uint32_t* qa_row = reinterpret_cast<const uint32_t*>(p.q + (token0 + tok_a) * p.q_token +
                                                                   (head0 + g - tok_a * group) * p.q_head);
        const uint32_t* qb_row = reinterpret_cast<const uint32_t*>(p.q + (token0 + tok_b) * p.q_token +
                                                                   (head0 + g + 8 - tok_b * group) * p.q_head);
        uint32_t qf[kSteps][4];
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
            qf[kk][0] = g < rows ? qa_row[kk * 8 + t] : 0u;
            qf[kk][1] = g + 8 < rows ? qb_row[kk * 8 + t] : 0u;
            qf[kk][2] = g < rows ? qa_row[kk * 8 + t + 4] : 0u;
            qf[kk][3] = g + 8 < rows ? qb_row[kk * 8 + t + 4] : 0u;
        }
        float o[kNTiles][4];
#pragma unroll
        for (int j = 0; j < kNTiles; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.0f, l_b = 0.0f;

        for (int i = 0; i < s.count; ++i, ++it) {
            const int slot = it % C::kStages;
            if (ok) ok = __all_sync(0xffffffffu, wait_paged(full(slot), (it / C::kStages) & 1, abort_flag, kSiteNarrowFull));
            const int key0 = (s.tile + i) * kNarrowKeys + warp * 16;
            if (ok && key0 < kv) {
                const uint32_t k_tile = base + slot * C::kStage, v_tile = k_tile + C::kTile;
                float sc[2][4] = {};
#pragma unroll
                for (int kk = 0; kk < kSteps; ++kk) {
                    uint32_t b[4];
                    ldmatrix_x4(k_tile + swizzled(k_row, 2 * kk + k_chunk), b);
                    mma_16816(sc[0], qf[kk], b[0], b[1]);
                    mma_16816(sc[1], qf[kk], b[2], b[3]);
                }
                if (key0 + 15 > first_limit) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int key = key0 + 8 * j + 2 * t + e;
                            if (key > limit_a) sc[j][e] = -INFINITY;
                            if (key > limit_b) sc[j][2 + e] = -INFINITY;
                        }
                }
                float top_a = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
                float top_b = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    top_a = fmaxf(top_a, __shfl_xor_sync(0xffffffffu, top_a, d));
                    top_b = fmaxf(top_b, __shfl_xor_sync(0xffffffffu, top_b, d));
                }
                // The base of a row's exponents moves only when a score exceeds it by a factor 2^16 (a weight
                // keeps its relative precision in bf16, sums are 32-bit), so O is rarely rescaled.
                const bool move_a = (top_a - m_a) * sl2 > kRebase, move_b = (top_b - m_b) * sl2 > kRebase;
                if (__any_sync(0xffffffffu, move_a || move_b)) {
                    const float keep_a = move_a ? ex2_approx((m_a - top_a) * sl2) : 1.0f;
                    const float keep_b = move_b ? ex2_approx((m_b - top_b) * sl2) : 1.0f;
                    if (move_a) m_a = top_a;
                    if (move_b) m_b = top_b;
                    l_a *= keep_a;
                    l_b *= keep_b;
#pragma unroll
                    for (int j = 0; j < kNTiles; ++j) {
                        o[j][0] *= keep_a;
                        o[j][1] *= keep_a;
                        o[j][2] *= keep_b;
                        o[j][3] *= keep_b;
                    }
                }
                const float base_a = m_a == -INFINITY ? 0.0f : m_a * sl2, base_b = m_b == -INFINITY ? 0.0f : m_b * sl2;
                uint32_t pf[4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float a0 = ex2_approx(fmaf(sc[j][0], sl2, -base_a)), a1 = ex2_approx(fmaf(sc[j][1], sl2, -base_a));
                    const float b0 = ex2_approx(fmaf(sc[j][2], sl2, -base_b)), b1 = ex2_approx(fmaf(sc[j][3], sl2, -base_b));
                    l_a += a0 + a1;
                    l_b += b0 + b1;
                    pf[2 * j] = pack_bf16x2(a0, a1);
                    pf[2 * j + 1] = pack_bf16x2(b0, b1);
                }
                // V rows behind the last key may hold anything: they are zeroed in the fragments (fragment
                // register 0 holds keys 2t and 2t + 1 of the 16, register 1 the same plus 8).
                uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
                const bool tail = key0 + 15 >= kv;
                if (tail) {
                    const int k0 = key0 + 2 * t;
                    keep0 = (k0 < kv ? 0xffffu : 0u) | (k0 + 1 < kv ? 0xffff0000u : 0u);
                    keep1 = (k0 + 8 < kv ? 0xffffu : 0u) | (k0 + 9 < kv ? 0xffff0000u : 0u);
                }
#pragma unroll
                for (int dd = 0; dd < kSteps; ++dd) {
                    uint32_t b[4];
                    ldmatrix_x4_trans(v_tile + swizzled(v_row, 2 * dd + v_chunk), b);
                    if (tail) {
                        b[0] &= keep0;
                        b[1] &= keep1;
                        b[2] &= keep0;
                        b[3] &= keep1;
                    }
                    mma_16816(o[2 * dd], pf, b[0], b[1]);
                    mma_16816(o[2 * dd + 1], pf, b[2], b[3]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(slot));
        }

        // ---- the four warps' results become one --------------------------------
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
            l_a += __shfl_xor_sync(0xffffffffu, l_a, d);
            l_b += __shfl_xor_sync(0xffffffffu, l_b, d);
        }
        if (t == 0) {
            stats[warp * 16 + g] = m_a;
            stats[warp * 16 + g + 8] = m_b;
            stats[64 + warp * 16 + g] = l_a;
            stats[64 + warp * 16 + g + 8] = l_b;
        }
        named_barrier(1, kNarrowWarps * 32);
        float all_a = -INFINITY, all_b = -INFINITY;
#pragma unroll
        for (int w = 0; w < kNarrowWarps; ++w) {
            all_a = fmaxf(all_a, stats[w * 16 + g]);
            all_b = fmaxf(all_b, stats[w * 16 + g + 8]);
        }
        float sum_a = 0.0f, sum_b = 0.0f, mine_a = 0.0f, mine_b = 0.0f;
#pragma unroll
        for (int w = 0; w < kNarrowWarps; ++w) {
            const float ma = stats[w * 16 + g], mb = stats[w * 16 + g + 8];
            const float wa = ma == -INFINITY ? 0.0f : ex2_approx((ma - all_a) * sl2);
            const float wb = mb == -INFINITY ? 0.0f : ex2_approx((mb - all_b) * sl2);
            sum_a += wa * stats[64 + w * 16 + g];
            sum_b += wb * stats[64 + w * 16 + g + 8];
            if (w == warp) { mine_a = wa; mine_b = wb; }
        }
        const bool whole = s.tile == 0 && s.tile + s.count == s.last - s.first;
        // An item that began before this CTA's range leaves its part in the CTA's first place, one that
        // goes on behind it in the second.
        float* part = p.partial + (2LL * blockIdx.x + (s.first < begin ? 0 : 1)) * C::kPartFloats;
        const float inv_a = whole ? 1.0f / sum_a : 1.0f, inv_b = whole ? 1.0f / sum_b : 1.0f;
        constexpr int kPer = kNTiles / 4;
#pragma unroll
        for (int quarter = 0; quarter < 4; ++quarter) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const float(&v)[4] = o[quarter * kPer + j];
                float* at = merge + (warp * 16 + g) * C::kMergeStride + 8 * j + 2 * t;
                *reinterpret_cast<float2*>(at) = make_float2(v[0] * mine_a, v[1] * mine_a);
                *reinterpret_cast<float2*>(at + 8 * C::kMergeStride) = make_float2(v[2] * mine_b, v[3] * mine_b);
            }
            named_barrier(1, kNarrowWarps * 32);
            if (warp == quarter) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    float2 a = make_float2(0.0f, 0.0f), b = a;
#pragma unroll
                    for (int w = 0; w < kNarrowWarps; ++w) {
                        const float* at = merge + (w * 16 + g) * C::kMergeStride + 8 * j + 2 * t;
                        const float2 va = *reinterpret_cast<const float2*>(at);
                        const float2 vb = *reinterpret_cast<const float2*>(at + 8 * C::kMergeStride);
                        a.x += va.x;
                        a.y += va.y;
                        b.x += vb.x;
                        b.y += vb.y;
                    }
                    const int column = quarter * C::kQuarter + 8 * j + 2 * t;
                    if (!ok) continue;
                    if (whole) {
                        if (g < rows)
                            *reinterpret_cast<uint32_t*>(p.o + (token0 + tok_a) * p.o_token +
                                                         (head0 + g - tok_a * group) * p.o_head + column) =
                                pack_bf16x2(a.x * inv_a, a.y * inv_a);
                        if (g + 8 < rows)
                            *reinterpret_cast<uint32_t*>(p.o + (token0 + tok_b) * p.o_token +
                                                         (head0 + g + 8 - tok_b * group) * p.o_head + column) =
                                pack_bf16x2(b.x * inv_b, b.y * inv_b);
                    } else {
                        if (g < rows) *reinterpret_cast<float2*>(part + g * D + column) = a;
                        if (g + 8 < rows) *reinterpret_cast<float2*>(part + (g + 8) * D + column) = b;
                    }
                }
            }
            named_barrier(1, kNarrowWarps * 32);
        }
        if (!whole && warp == 0 && t == 0) {
            part[16 * D + g] = all_a;
            part[16 * D + g + 8] = all_b;
            part[16 * D + 16 + g] = sum_a;
            part[16 * D + 16 + g + 8] = sum_b;
        }
    }
}

// One block per border between two CTAs' ranges; the first border inside an item merges the item's
// parts, in their order, one warp per row.
template <int D>
__global__ void __launch_bounds__(kNarrowRows * 32)
combine_narrow_kernel(const __grid_constant__ PagedParams p, int ctas)
{
    using C = NarrowCfg<D>;
    const FaPagedPlan& plan = p.plan;
    const long long* start = narrow_starts(plan.schedule, plan.num_seqs);
    const long long total = start[plan.num_seqs] * plan.kv_heads;
    const long long share = narrow_share(total, ctas);
    const long long border = share * (blockIdx.x + 1);
    if (border >= total) return;
    const NarrowSegment s = narrow_segment(plan, start, border, total);
    if (s.first == border || s.first < border - share) return;
    const int row = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int token0 = plan.query_start[s.b], n = plan.query_start[s.b + 1] - token0;
    const int group = plan.heads / plan.kv_heads;
    if (row >= n * group) return;
    const long long c0 = s.first / share, c1 = (s.last - 1) / share;
    // The first part ends its CTA's range; the others begin theirs.
    auto part = [&](long long c) { return p.partial + (2 * c + (c == c0 ? 1 : 0)) * C::kPartFloats; };
    float top = -INFINITY;
    for (long long c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, part(c)[16 * D + row]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    constexpr int E = D / 32;
    float acc[E] = {}, sum = 0.0f;
#pragma unroll 4
    for (long long c = c0; c <= c1; ++c) {
        const float* at = part(c);
        const float m = at[16 * D + row];
        const float w = m == -INFINITY ? 0.0f : ex2_approx((m - top) * p.scale_log2);
        sum += w * at[16 * D + 16 + row];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += w * at[row * D + lane * E + e];
    }
    const float inv = 1.0f / sum;
    const int tok = row / group;
    __nv_bfloat16* out = p.o + (token0 + tok) * p.o_token + (s.h * group + row - tok * group) * p.o_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2)
        *reinterpret_cast<uint32_t*>(out + e) = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
}

// One warp per query row: a lane holds D / 32 elements of q and of the accumulator.
template <int D>
__global__ void __launch_bounds__(128)
paged_rows_kernel(const PagedParams p)
{
    constexpr int E = D / 32;
    const FaPagedPlan& plan = p.plan;
    const int lane = threadIdx.x % 32;
    const long long row = (static_cast<long long>(blockIdx.x) * 128 + threadIdx.x) / 32;
    const int token = static_cast<int>(row / plan.heads);
    const int head = static_cast<int>(row % plan.heads);
    if (token >= plan.query_start[plan.num_seqs]) return;
    int lo = 0, hi = plan.num_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (plan.query_start[mid] <= token) lo = mid;
        else hi = mid - 1;
    }
    const int start = plan.query_start[lo], n = plan.query_start[lo + 1] - start, kv = plan.kv_lens[lo];
    if (kv < n || n * (plan.heads / plan.kv_heads) <= kNarrowRows) return;
    const int keys = plan.causal ? kv - n + (token - start) + 1 : kv;
    const int kv_head = head / (plan.heads / plan.kv_heads);
    float q[E], acc[E] = {}, m = -INFINITY, l = 0.0f;
    for (int e = 0; e < E; ++e) q[e] = __bfloat162float(p.q[token * p.q_token + head * p.q_head + lane * E + e]);
    for (int j = 0; j < keys; ++j) {
        const int page = plan.block_table[static_cast<long long>(lo) * plan.table_stride + (j >> p.page_shift)];
        if (page < 0 || page >= plan.num_pages) {
            atomicOr(&g_paged_error_word, FA_ERROR_BAD_PAGE);
            return;
        }
        const int r = j & ((1 << p.page_shift) - 1);
        const __nv_bfloat16* k = p.k + page * p.k_page + kv_head * p.k_head + r * p.k_row + lane * E;
        const __nv_bfloat16* v = p.v + page * p.v_page + kv_head * p.v_head + r * p.v_row + lane * E;
        float dot = 0.0f;
        for (int e = 0; e < E; ++e) dot += q[e] * __bfloat162float(k[e]);
        for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        const float s = dot * p.scale_log2;
        const float top = fmaxf(m, s);
        const float keep = exp2f(m - top), w = exp2f(s - top);
        l = l * keep + w;
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * keep + w * __bfloat162float(v[e]);
        m = top;
    }
    for (int e = 0; e < E; ++e)
        p.o[token * p.o_token + head * p.o_head + lane * E + e] = __float2bfloat16_rn(acc[e] / l);
}

}  // namespace fa_sm100

// =============================================================================
// Host side
// =============================================================================
namespace fa_sm100_internal {

bool page_size_supported(int page_size)
{
    return page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0;
}

int current_sm100(int* device, int* sm_count)
{
    constexpr int kMax = 64;
    static int counts[kMax];        // SM count of each device once known (written with the same value by any thread)
    cudaError_t err = cudaGetDevice(device);
    if (err != cudaSuccess) return static_cast<int>(err);
    if (*device < 0 || *device >= kMax) return FA_STATUS_INVALID_ARGUMENT;
    if (counts[*device] == 0) {
        int major = 0, count = 0;
        err = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *device);
        if (err != cudaSuccess) return static_cast<int>(err);
        if (major != 10) return FA_STATUS_NO_SM100;
        err = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, *device);
        if (err != cudaSuccess) return static_cast<int>(err);
        counts[*device] = count;
    }
    *sm_count = counts[*device];
    return FA_STATUS_OK;
}

int validate_plan(const FaPagedPlan* plan)
{
    if (plan == nullptr) return FA_STATUS_INVALID_ARGUMENT;
    if (plan->head_dim != 64 && plan->head_dim != 128) return FA_STATUS_UNSUPPORTED;
    if (!page_size_supported(plan->page_size)) return FA_STATUS_UNSUPPORTED;
    if (plan->heads < 1 || plan->kv_heads < 1 || plan->heads % plan->kv_heads) return FA_STATUS_INVALID_ARGUMENT;
    if (plan->heads / plan->kv_heads > 128) return FA_STATUS_UNSUPPORTED;
    if (plan->num_seqs < 0 || plan->total_tokens < 0 || plan->max_new < 0 || plan->num_pages < 0 ||
        plan->table_width < 0 || plan->table_stride < plan->table_width)
        return FA_STATUS_INVALID_ARGUMENT;
    if (static_cast<long long>(plan->num_pages) * plan->page_size > INT_MAX ||
        static_cast<long long>(plan->table_width) * plan->page_size > INT_MAX)
        return FA_STATUS_INVALID_ARGUMENT;
    if (plan->query_start == nullptr || plan->free_cursor == nullptr || plan->schedule == nullptr)
        return FA_STATUS_INVALID_ARGUMENT;
    if (plan->num_seqs > 0 && (plan->kv_lens == nullptr || (plan->table_width > 0 && plan->block_table == nullptr)))
        return FA_STATUS_INVALID_ARGUMENT;
    if (plan->total_tokens > 0 && (plan->positions == nullptr || plan->slots == nullptr))
        return FA_STATUS_INVALID_ARGUMENT;
    return FA_STATUS_OK;
}

int take_paged_attention_error(unsigned int* word)
{
    cudaError_t err = cudaMemcpyFromSymbol(word, fa_sm100::g_paged_error_word, sizeof(*word));
    const unsigned int zero = 0;
    if (err == cudaSuccess && *word != 0) err = cudaMemcpyToSymbol(fa_sm100::g_paged_error_word, &zero, sizeof(zero));
    return static_cast<int>(err);
}

}  // namespace fa_sm100_internal

namespace {

using namespace fa_sm100;

// The kernels' shared-memory opt-in, once per device.
struct PagedDevice {
    std::once_flag once;
    int status = FA_STATUS_OK;
};
PagedDevice g_paged_devices[64];

int prepare_paged_device(int device)
{
    PagedDevice& state = g_paged_devices[device];
    std::call_once(state.once, [&]() {
        cudaError_t err = cudaFuncSetAttribute(reinterpret_cast<const void*>(paged_narrow_kernel<64>),
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, NarrowCfg<64>::kSmemBytes);
        if (err == cudaSuccess)
            err = cudaFuncSetAttribute(reinterpret_cast<const void*>(paged_narrow_kernel<128>),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, NarrowCfg<128>::kSmemBytes);
        state.status = static_cast<int>(err);
    });
    return state.status;
}

int narrow_ctas(int sms) { return kNarrowCtasPerSm * sms; }

size_t narrow_workspace(int sms, int head_dim)
{
    return static_cast<size_t>(narrow_ctas(sms)) * 2 * kNarrowRows * (head_dim + 2) * sizeof(float);
}

// A cache as [page][head][row][D]: boxes of 64 columns by `rows` rows of one head of one page.
int cache_map(CUtensorMap* map, const void* ptr, const FaPagedPlan& plan, const long long* strides, int rows)
{
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(plan.head_dim), static_cast<cuuint64_t>(plan.page_size),
                                static_cast<cuuint64_t>(plan.kv_heads), static_cast<cuuint64_t>(plan.num_pages)};
    const cuuint64_t bytes[3] = {static_cast<cuuint64_t>(strides[2]) * 2u, static_cast<cuuint64_t>(strides[1]) * 2u,
                                 static_cast<cuuint64_t>(strides[0]) * 2u};
    const cuuint32_t box[4] = {64u, static_cast<cuuint32_t>(plan.page_size < rows ? plan.page_size : rows), 1u, 1u};
    return fa_sm100_internal::encode_map(map, ptr, 4, dims, bytes, box);
}

template <int D>
int launch_narrow(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const PagedParams& params, int sms, cudaStream_t stream)
{
    const int ctas = narrow_ctas(sms);
    paged_narrow_kernel<D><<<ctas, kNarrowThreads, NarrowCfg<D>::kSmemBytes, stream>>>(tm_k, tm_v, params);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return static_cast<int>(err);
    combine_narrow_kernel<D><<<ctas - 1, kNarrowRows * 32, 0, stream>>>(params, ctas);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace

extern "C" {

size_t fa_sm100_paged_workspace_bytes(const FaPagedPlan* plan)
{
    int device = 0, sms = 0;
    if (fa_sm100_internal::validate_plan(plan) != FA_STATUS_OK ||
        fa_sm100_internal::current_sm100(&device, &sms) != FA_STATUS_OK)
        return 0;
    return narrow_workspace(sms, plan->head_dim);
}

int fa_sm100_paged_fwd(const FaPagedPlan* plan, const void* q, const void* k_cache, const void* v_cache, void* o,
                       const long long* strides, void* workspace, size_t workspace_bytes, void* stream)
{
    using namespace fa_sm100;
    int status = fa_sm100_internal::validate_plan(plan);
    if (status != FA_STATUS_OK) return status;
    if (strides == nullptr) return FA_STATUS_INVALID_ARGUMENT;
    if (plan->total_tokens == 0 || plan->num_seqs == 0) return FA_STATUS_OK;
    if (q == nullptr || k_cache == nullptr || v_cache == nullptr || o == nullptr) return FA_STATUS_INVALID_ARGUMENT;
    uintptr_t any = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) |
                    reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(o);
    if (any & 15u) return FA_STATUS_MISALIGNED;
    for (int i = 0; i < 10; ++i)
        if (strides[i] & 7) return FA_STATUS_MISALIGNED;
    int device = 0, sms = 0;
    status = fa_sm100_internal::current_sm100(&device, &sms);
    if (status != FA_STATUS_OK) return status;
    if ((status = prepare_paged_device(device)) != FA_STATUS_OK) return status;
    if (workspace_bytes < narrow_workspace(sms, plan->head_dim)) return FA_STATUS_WORKSPACE;
    if (workspace == nullptr || plan->num_pages == 0) return FA_STATUS_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return FA_STATUS_MISALIGNED;
    PagedParams params{};
    params.plan = *plan;
    params.q = static_cast<const __nv_bfloat16*>(q);
    params.k = static_cast<const __nv_bfloat16*>(k_cache);
    params.v = static_cast<const __nv_bfloat16*>(v_cache);
    params.o = static_cast<__nv_bfloat16*>(o);
    params.q_token = strides[0];
    params.q_head = strides[1];
    params.o_token = strides[2];
    params.o_head = strides[3];
    params.k_page = strides[4];
    params.k_head = strides[5];
    params.k_row = strides[6];
    params.v_page = strides[7];
    params.v_head = strides[8];
    params.v_row = strides[9];
    params.page_shift = __builtin_ctz(static_cast<unsigned>(plan->page_size));
    params.scale_log2 = fa_default_scale(plan->head_dim) * 1.4426950408889634f;
    params.partial = static_cast<float*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    CUtensorMap tm_k, tm_v;
    if ((status = cache_map(&tm_k, k_cache, *plan, strides + 4, kNarrowKeys)) != FA_STATUS_OK) return status;
    if ((status = cache_map(&tm_v, v_cache, *plan, strides + 7, kNarrowKeys)) != FA_STATUS_OK) return status;
    status = plan->head_dim == 64 ? launch_narrow<64>(tm_k, tm_v, params, sms, s)
                                  : launch_narrow<128>(tm_k, tm_v, params, sms, s);
    if (status != FA_STATUS_OK) return status;
    const long long rows = static_cast<long long>(plan->total_tokens) * plan->heads;
    const long long blocks = (rows + 3) / 4;
    if (blocks > INT_MAX) return FA_STATUS_INVALID_ARGUMENT;
    if (plan->head_dim == 64) paged_rows_kernel<64><<<static_cast<unsigned>(blocks), 128, 0, s>>>(params);
    else paged_rows_kernel<128><<<static_cast<unsigned>(blocks), 128, 0, s>>>(params);
    return static_cast<int>(cudaGetLastError());
}

}  // extern "C"
