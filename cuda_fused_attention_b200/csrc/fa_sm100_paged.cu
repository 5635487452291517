// Attention of a step's new tokens over a paged K/V cache (sm_100a).

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
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
    __nv_bfloat16* o;
    long long q_token, q_head, o_token, o_head;     // K and V are read through tensor maps
    int page_shift;
    float scale_log2;
    int behind_wide;            // narrow kernel: the wide one of the same call was launched before it
    int narrow_follows;         // wide kernel: the narrow one of the same call is launched behind it
    int inject_stall;           // test only: the warps that hand out work wait on a barrier nothing arrives on
    // Parts of items that cross a border between CTAs' ranges, two places per CTA, and per CTA what is to be
    // merged from the second place on; for the narrow and for the wide kernel.
    float* partial;
    struct Merge* merges;
    float* wide_partial;
    struct Merge* wide_merges;
};

// The item whose first part lies in a CTA's second place: it has `parts` parts, the others in the first
// places of the CTAs that follow. 0: there is none.
struct Merge {
    int parts;
    int token0, tokens, head0;      // packed row of the first token, tokens, first query head
};

// A row keeps its exponent base until a score exceeds it by this much in the exp2 domain.
constexpr float kRebase = 16.0f;

// =============================================================================
// Narrow kernel: requests of few query rows per K/V head (decode steps, drafted tokens)
// =============================================================================
// Each K/V byte is used for at most 32 rows, so the cache's bytes bound it: 512 bytes a key at
// D = 128 against 32 * 4 * 128 operations. The work of all requests and K/V heads is one line of
// 64-key tiles (request, then head, then key; each item preceded by kNarrowGap idle units that stand
// for its set-up), and each of the grid's CTAs (two per SM) takes an equal stretch of it, whatever the
// requests' lengths: an item that crosses a border is merged from parts (paged_combine_narrow_kernel). A
// CTA's warp 4 streams the tiles by TMA through a ring that runs on across items, page by page (a page
// that is absent reads as zeros), with each item's Q and description ahead of its first tile; warps
// 0-3 share out the keys of every tile (and the two 16-row tiles, if MT, their number, is 2), S = Q K^T
// and O += P V by warp-level matrix instructions with Q, P and O in registers, a running maximum and
// sum per warp, and meet only at an item's end, in the ring slot of its last tile. P goes into the
// product with V as two bf16 numbers (rounded, and the rest), so that it keeps 16 bits; everything
// else that is kept is 32-bit. Why mma.sync and not tcgen05: a tile of 128 rows would be nearly empty, and
// its fragments keep up with memory. Measured (B200, 32/8 heads, D = 128): 64 requests of 4095 to
// 16384 keys 410 us, 6.6 TB/s; 32 of up to 4096 keys 52 us with the merging, 5.3 TB/s; 16 of 5 to 8
// new tokens behind up to 8192 (MT = 2) 62 to 66 us, 4.6 to 4.9 TB/s, and 69 us a call.
constexpr int kNarrowWarps = 4;
constexpr int kNarrowThreads = (kNarrowWarps + 1) * 32;
constexpr int kNarrowCtasPerSm = 2;
constexpr int kNarrowMinTiles = 2;       // units a CTA takes at least (2048 keys, 8 heads: 8.5 us; 3: 8.8, 5: 10.5, 8: 11.5)
constexpr unsigned long long kTimeoutNs = 1000000000ull;

// What the producer tells the consumers of a stretch of one (request, K/V head).
struct NarrowItem {
    int token0, tokens, head0, kv;      // packed row of the first token, tokens, first query head, keys
    int tile, count;                    // key tiles [tile, tile + count); count 0 ends the walk
    int part;                           // place of its part, -1: the whole item, written directly
    int reserved;
};

template <int D, int MT>
struct NarrowCfg {
    static constexpr int kTile = kNarrowKeys * D * 2;               // bytes of a K or V tile
    static constexpr int kStage = 2 * kTile;
    static constexpr int kStages = D == 128 ? 3 : 6;                // 96 KB in flight per CTA
    static constexpr int kQSlots = D == 128 ? (MT == 1 ? 3 : 1) : (MT == 1 ? 4 : 2);    // as many as fit
    static constexpr int kQStride = 2 * D + 16;                     // bytes; the pad spreads rows over banks
    static constexpr int kQBytes = 16 * MT * kQStride;
    static constexpr int kQOff = kStages * kStage;
    static constexpr int kStatsOff = kQOff + kQSlots * kQBytes;     // [key group][row] maxima, then sums
    static constexpr int kStats = kNarrowWarps * 16;
    static constexpr int kItemOff = kStatsOff + 2 * kStats * 4;
    static constexpr int kBarOff = kItemOff + kQSlots * static_cast<int>(sizeof(NarrowItem));
    static constexpr int kNumBars = 2 * kStages + 2 * kQSlots;
    static constexpr int kAbortOff = kBarOff + kNumBars * 8;
    static constexpr int kSmemBytes = kAbortOff + 16 + 1024;        // slack for 1024-byte alignment
    static constexpr int kPartFloats = 16 * MT * (D + 2);           // O [rows][D], maxima, sums
    static_assert(kNarrowWarps * 16 * D * 4 == kStage, "a merge fits one ring slot");
    static_assert(2 * (kSmemBytes + 1024) <= 233472, "two CTAs per SM");
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

enum PagedSite : uint32_t { kSiteNarrowFull = 32, kSiteNarrowEmpty = 33, kSiteNarrowItem = 34, kSiteNarrowItemFree = 35 };

// A request as the attention kernels see it: the units of one K/V head on the line, and its tokens and keys.
struct Request {
    int b;
    long long start, units;
    int token0, tokens, kv;
};

// Finds requests by their place on the line, for one warp (all lanes with the same arguments). Up to 32 requests
// are held in the lanes, loaded together when the kernel starts; with more, 32 borders are read at a time, so a
// thousand requests take two round trips to memory.
class RequestFinder {
public:
    __device__ __forceinline__ RequestFinder(const FaPagedPlan& plan, const long long* start)
        : plan_(plan), start_(start), lane_(threadIdx.x % 32), held_(plan.num_seqs <= 32)
    {
        if (held_ && lane_ < plan.num_seqs) {
            my_start_ = start[lane_];
            my_end_ = start[lane_ + 1];
            my_token0_ = plan.query_start[lane_];
            my_tokens_ = plan.query_start[lane_ + 1] - my_token0_;
            my_kv_ = plan.kv_lens[lane_];
        }
    }
    // The request whose units [start, start + units) hold y.
    __device__ __forceinline__ Request find(long long y) const
    {
        Request r;
        if (held_) {
            r.b = last_of(lane_ < plan_.num_seqs && my_start_ <= y);
            r.start = __shfl_sync(0xffffffffu, my_start_, r.b);
            r.units = __shfl_sync(0xffffffffu, my_end_, r.b) - r.start;
            r.token0 = __shfl_sync(0xffffffffu, my_token0_, r.b);
            r.tokens = __shfl_sync(0xffffffffu, my_tokens_, r.b);
            r.kv = __shfl_sync(0xffffffffu, my_kv_, r.b);
            return r;
        }
        int lo = 0, count = plan_.num_seqs;         // the last request in [lo, lo + count) that begins at or before y
        while (count > 1) {
            const int step = (count + 31) / 32;
            const int at = last_of(lane_ * step < count && start_[lo + lane_ * step] <= y);
            lo += at * step;
            count = min(step, count - at * step);
        }
        r.b = lo;
        r.start = start_[lo];
        r.units = start_[lo + 1] - r.start;
        r.token0 = plan_.query_start[lo];
        r.tokens = plan_.query_start[lo + 1] - r.token0;
        r.kv = plan_.kv_lens[lo];
        return r;
    }
    // The last lane for which the condition holds (it does for lane 0).
    static __device__ __forceinline__ int last_of(bool condition)
    {
        return 31 - __clz(static_cast<int>(__ballot_sync(0xffffffffu, condition)));
    }

private:
    const FaPagedPlan& plan_;
    const long long* start_;
    const int lane_;
    const bool held_;
    long long my_start_ = 0, my_end_ = 0;
    int my_token0_ = 0, my_tokens_ = 0, my_kv_ = 0;
};

// The plan's arrays may have been written again for other arguments (mask, max_new, table) than a captured call was
// made with. Its line of units is then another one, and to walk it might never end or leave the tensors: what a
// kernel finds on the line is compared with its own arguments, and a difference ends the walk.
__device__ __forceinline__ void record_other_plan() { atomicOr(&g_paged_error_word, FA_ERROR_OTHER_PLAN); }

__device__ __forceinline__ bool request_in_range(const FaPagedPlan& plan, const Request& r)
{
    return r.token0 >= 0 && r.tokens > 0 && r.tokens <= plan.total_tokens - r.token0 && r.kv > 0 &&
           r.kv <= plan.table_width * plan.page_size;
}

// Units per CTA when `total` are shared out over `ctas`.
__device__ __forceinline__ long long narrow_share(long long total, int ctas)
{
    const long long even = ceil_div(total, ctas);
    return even > kNarrowMinTiles ? even : kNarrowMinTiles;
}

template <int D, int MT>
__global__ void __launch_bounds__(kNarrowThreads, kNarrowCtasPerSm)
paged_narrow_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ PagedParams p)
{
    using C = NarrowCfg<D, MT>;
    const FaPagedPlan& plan = p.plan;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int group = plan.heads / plan.kv_heads;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + C::kAbortOff);
    NarrowItem* items = reinterpret_cast<NarrowItem*>(smem + C::kItemOff);
    auto bar = [&](int i) -> uint32_t { return base + C::kBarOff + static_cast<uint32_t>(i) * 8u; };
    auto full = [&](int s) -> uint32_t { return bar(s); };
    auto empty = [&](int s) -> uint32_t { return bar(C::kStages + s); };
    auto item_full = [&](int s) -> uint32_t { return bar(2 * C::kStages + s); };
    auto item_empty = [&](int s) -> uint32_t { return bar(2 * C::kStages + C::kQSlots + s); };
    if (warp == 0) {
        for (int i = lane; i < C::kNumBars; i += 32) {
            const bool released = (i >= C::kStages && i < 2 * C::kStages) || i >= 2 * C::kStages + C::kQSlots;
            mbar_init(bar(i), released ? kNarrowWarps : 1);
        }
        if (lane == 0) *abort_flag = 0u;
        fence_mbarrier_init();
    }
    // Behind the wide kernel of the same call, which has waited, there is nothing to wait for before the end.
    if (!p.behind_wide) grid_dependency_wait();
    grid_dependents_launch();
    const long long* start = narrow_starts(plan.schedule);
    const long long total = start[plan.num_seqs] * plan.kv_heads;
    const RequestFinder finder(plan, start);        // used by the producer
    const long long share = narrow_share(total, gridDim.x);
    const long long begin = share * blockIdx.x;
    // By one thread: work for a wide kernel that this call has none of.
    auto check_wide = [&]() {
        if (blockIdx.x == 0 && !p.behind_wide && wide_starts(plan.schedule, plan.num_seqs)[plan.num_seqs] != 0) record_other_plan();
    };
    if (begin >= total) {
        if (threadIdx.x == 0) {
            check_wide();
            p.merges[blockIdx.x] = Merge{};
        }
        grid_dependency_wait();
        return;
    }
    const long long end = begin + share < total ? begin + share : total;
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
        int it = 0, sg = 0;
        Merge merge{};
        bool ok = p.inject_stall == 0 || __all_sync(0xffffffffu, wait_paged(item_empty(0), 0, abort_flag, kSiteNarrowItemFree));
        for (long long x = begin; ok;) {
            NarrowItem item{};
            int b = 0, h = 0;
            if (x < end) {
                const Request r = finder.find(quotient(x, plan.kv_heads));
                if (!request_in_range(plan, r) || r.tokens * static_cast<long long>(group) > 16 * MT ||
                    r.units != kNarrowGap + (r.kv + kNarrowKeys - 1) / kNarrowKeys) {
                    if (lane == 0) record_other_plan();
                    x = end;
                    continue;
                }
                b = r.b;
                h = static_cast<int>(quotient(x - r.start * plan.kv_heads, r.units));
                // The item's tiles lie at [first, last) of the line, behind its gap.
                const long long first = r.start * plan.kv_heads + h * r.units + kNarrowGap;
                const long long last = first - kNarrowGap + r.units;
                if (x < first) x = first;
                const long long stop = last < end ? last : end;
                if (x >= stop) {                // only idle units are left of this range
                    x = last;
                    continue;
                }
                item.token0 = r.token0;
                item.tokens = r.tokens;
                item.head0 = h * group;
                item.kv = r.kv;
                item.tile = static_cast<int>(x - first);
                item.count = static_cast<int>(stop - x);
                // An item that began before this CTA's range leaves its part in the CTA's first place, one that
                // goes on behind it in the second.
                item.part = first < begin ? 2 * static_cast<int>(blockIdx.x)
                                          : last > end ? 2 * static_cast<int>(blockIdx.x) + 1 : -1;
                if (first >= begin && last > end)
                    merge = {static_cast<int>(quotient(last - 1, share)) - static_cast<int>(blockIdx.x) + 1, item.token0, item.tokens,
                             item.head0};
                x = stop;
            }
            const int q_slot = sg % C::kQSlots;
            if (sg >= C::kQSlots && !__all_sync(0xffffffffu, wait_paged(item_empty(q_slot), (sg / C::kQSlots - 1) & 1, abort_flag,
                                                                         kSiteNarrowItemFree))) {
                ok = false;
                break;
            }
            const int q_rows = item.count > 0 ? item.tokens * group : 0;
            if (lane == 0) {
                items[q_slot] = item;
                mbar_arrive_expect_tx(item_full(q_slot), static_cast<uint32_t>(q_rows * 2 * D));
            }
            __syncwarp();
            ++sg;
            if (item.count == 0) break;
            if (lane < q_rows) {
                const int tok = lane / group;
                bulk_load(base + C::kQOff + q_slot * C::kQBytes + lane * C::kQStride,
                          p.q + (item.token0 + tok) * p.q_token + (item.head0 + lane - tok * group) * p.q_head, 2 * D,
                          item_full(q_slot));
            }
            const int* table = plan.block_table + static_cast<long long>(b) * plan.table_stride;
            const int held = (item.kv + plan.page_size - 1) >> p.page_shift;
            auto page_at = [&](int tile) -> int {
                // num_pages is out of the map's range: such a box reads as zeros.
                const int i = ((tile * kNarrowKeys) >> p.page_shift) + page_of_tile;
                if (!active || i >= held) return plan.num_pages;
                const int page = table[i];     // an ordinary load: the plan may have been written while this CTA was here
                if (page >= 0 && page < plan.num_pages) return page;
                atomicOr(&g_paged_error_word, FA_ERROR_BAD_PAGE);
                return plan.num_pages;
            };
            int page = page_at(item.tile);
            for (int i = 0; i < item.count; ++i, ++it) {
                const int slot = it % C::kStages, use = it / C::kStages;
                const int row = ((item.tile + i) * kNarrowKeys) & (plan.page_size - 1);
                if (use > 0 && !__all_sync(0xffffffffu, wait_paged(empty(slot), (use - 1) & 1, abort_flag, kSiteNarrowEmpty))) {
                    ok = false;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(full(slot), C::kStage);
                __syncwarp();
                if (active)
                    tma_load_4d(base + slot * C::kStage + offset, map, full(slot), block * 64, pages > 1 ? 0 : row, h, page);
                if (i + 1 < item.count) page = page_at(item.tile + i + 1);
            }
        }
        if (!ok && lane == 0) {
            for (int i = it > C::kStages ? it - C::kStages : 0; i < it; ++i) drain_paged(full(i % C::kStages), (i / C::kStages) & 1);
            for (int i = sg > C::kQSlots ? sg - C::kQSlots : 0; i < sg; ++i)
                drain_paged(item_full(i % C::kQSlots), (i / C::kQSlots) & 1);
        }
        if (lane == 0) {
            p.merges[blockIdx.x] = merge;
            check_wide();
        }
        grid_dependency_wait();     // what was launched before this kernel is done when this one is
        return;
    }

    // ======================= consumers =========================================
    // Warp (kg, mt) takes 16 * MT keys of each tile for 16 query rows. A warp that gave up (ok false) still
    // walks on, so that the others' barriers complete; nothing waits then.
    constexpr int kSteps = D / 16;
    constexpr int kNTiles = D / 8;
    constexpr int kGroups = kNarrowWarps / MT;      // warps that share out a tile's keys
    constexpr int kKeys = kNarrowKeys / kGroups;    // keys of a warp, 16 * MT
    float* stats = reinterpret_cast<float*>(smem + C::kStatsOff);
    const int mt = warp % MT, kg = warp / MT;
    const int g = lane >> 2, t = lane & 3;
    const float sl2 = p.scale_log2;
    // ldmatrix rows of this lane within a tile.
    const int k_row = kg * kKeys + (lane & 7) + ((lane >> 4) & 1) * 8, k_chunk = (lane >> 3) & 1;
    const int v_row = kg * kKeys + (lane & 7) + ((lane >> 3) & 1) * 8, v_chunk = (lane >> 4) & 1;
    auto swizzled = [](int row, int chunk) -> uint32_t {
        return static_cast<uint32_t>((chunk >> 3) * kNarrowKeys * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
    };
    int it = 0;
    bool ok = true;
    for (int sg = 0;; ++sg) {
        const int q_slot = sg % C::kQSlots;
        if (ok) ok = __all_sync(0xffffffffu, wait_paged(item_full(q_slot), (sg / C::kQSlots) & 1, abort_flag, kSiteNarrowItem));
        // All four warps leave together, or none.
        if (!named_barrier_and(1, kNarrowWarps * 32, ok)) break;
        const NarrowItem item = items[q_slot];
        if (item.count == 0) break;
        const int rows = item.tokens * group;
        const bool busy = 16 * mt < rows;           // this warp has rows
        uint32_t qf[kSteps][4];
        const uint32_t q_addr = base + C::kQOff + q_slot * C::kQBytes +
                                static_cast<uint32_t>((16 * mt + (lane & 7) + ((lane >> 3) & 1) * 8) * C::kQStride + (lane >> 4) * 16);
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) ldmatrix_x4(q_addr + kk * 32, qf[kk]);
        __syncwarp();
        if (lane == 0) mbar_arrive(item_empty(q_slot));
        const int first_limit = plan.causal ? item.kv - item.tokens : item.kv - 1;
        // Last keys of rows g and g + 8.
        const int limit0 = plan.causal ? first_limit + (16 * mt + g) / group : first_limit;
        const int limit1 = plan.causal ? first_limit + (16 * mt + 8 + g) / group : first_limit;
        float o[kNTiles][4];
#pragma unroll
        for (int j = 0; j < kNTiles; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

        for (int i = 0; i < item.count; ++i, ++it) {
            const int slot = it % C::kStages;
            if (ok) ok = __all_sync(0xffffffffu, wait_paged(full(slot), (it / C::kStages) & 1, abort_flag, kSiteNarrowFull));
            const int key0 = (item.tile + i) * kNarrowKeys + kg * kKeys;
            if (ok && busy && key0 < item.kv) {
                const uint32_t k_tile = base + slot * C::kStage, v_tile = k_tile + C::kTile;
                float sc[2 * MT][4] = {};
#pragma unroll
                for (int kk = 0; kk < kSteps; ++kk)
#pragma unroll
                    for (int s = 0; s < MT; ++s) {
                        uint32_t b[4];
                        ldmatrix_x4(k_tile + swizzled(k_row + 16 * s, 2 * kk + k_chunk), b);
                        mma_16816(sc[2 * s], qf[kk], b[0], b[1]);
                        mma_16816(sc[2 * s + 1], qf[kk], b[2], b[3]);
                    }
                if (key0 + kKeys - 1 > first_limit) {
#pragma unroll
                    for (int j = 0; j < 2 * MT; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int key = key0 + 8 * j + 2 * t + e;
                            if (key > limit0) sc[j][e] = -INFINITY;
                            if (key > limit1) sc[j][2 + e] = -INFINITY;
                        }
                }
                float top0 = fmaxf(sc[0][0], sc[0][1]), top1 = fmaxf(sc[0][2], sc[0][3]);
#pragma unroll
                for (int j = 1; j < 2 * MT; ++j) {
                    top0 = fmaxf(top0, fmaxf(sc[j][0], sc[j][1]));
                    top1 = fmaxf(top1, fmaxf(sc[j][2], sc[j][3]));
                }
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, d));
                    top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, d));
                }
                // The base of a row's exponents moves only when a score exceeds it by a factor 2^16 (a weight
                // keeps its relative precision in bf16, sums are 32-bit), so O is rarely rescaled.
                const bool move0 = (top0 - m0) * sl2 > kRebase, move1 = (top1 - m1) * sl2 > kRebase;
                if (__any_sync(0xffffffffu, move0 || move1)) {
                    const float keep0 = move0 ? ex2_approx((m0 - top0) * sl2) : 1.0f;
                    const float keep1 = move1 ? ex2_approx((m1 - top1) * sl2) : 1.0f;
                    if (move0) m0 = top0;
                    if (move1) m1 = top1;
                    l0 *= keep0;
                    l1 *= keep1;
#pragma unroll
                    for (int j = 0; j < kNTiles; ++j) {
                        o[j][0] *= keep0;
                        o[j][1] *= keep0;
                        o[j][2] *= keep1;
                        o[j][3] *= keep1;
                    }
                }
                const float base0 = m0 == -INFINITY ? 0.0f : m0 * sl2, base1 = m1 == -INFINITY ? 0.0f : m1 * sl2;
                // A weight as two bf16 numbers, rounded and rest: V's product is not bound by them, so P keeps 16 bits.
                uint32_t pf[MT][4], rest[MT][4];
#pragma unroll
                for (int j = 0; j < 2 * MT; ++j) {
                    const float a0 = ex2_approx(fmaf(sc[j][0], sl2, -base0)), a1 = ex2_approx(fmaf(sc[j][1], sl2, -base0));
                    const float b0 = ex2_approx(fmaf(sc[j][2], sl2, -base1)), b1 = ex2_approx(fmaf(sc[j][3], sl2, -base1));
                    l0 += a0 + a1;
                    l1 += b0 + b1;
                    const uint32_t a = pack_bf16x2(a0, a1), b = pack_bf16x2(b0, b1);
                    pf[j / 2][2 * (j % 2)] = a;
                    pf[j / 2][2 * (j % 2) + 1] = b;
                    rest[j / 2][2 * (j % 2)] = pack_bf16x2(a0 - __uint_as_float(a << 16), a1 - __uint_as_float(a & 0xffff0000u));
                    rest[j / 2][2 * (j % 2) + 1] = pack_bf16x2(b0 - __uint_as_float(b << 16), b1 - __uint_as_float(b & 0xffff0000u));
                }
                // V rows behind the last key may hold anything: they are zeroed in the fragments (fragment
                // register 0 holds keys 2t and 2t + 1 of 16, register 1 the same plus 8).
                const bool tail = key0 + kKeys > item.kv;
#pragma unroll
                for (int s = 0; s < MT; ++s) {
                    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
                    if (tail) {
                        const int k0 = key0 + 16 * s + 2 * t;
                        keep0 = (k0 < item.kv ? 0xffffu : 0u) | (k0 + 1 < item.kv ? 0xffff0000u : 0u);
                        keep1 = (k0 + 8 < item.kv ? 0xffffu : 0u) | (k0 + 9 < item.kv ? 0xffff0000u : 0u);
                    }
#pragma unroll
                    for (int dd = 0; dd < kSteps; ++dd) {
                        uint32_t b[4];
                        ldmatrix_x4_trans(v_tile + swizzled(v_row + 16 * s, 2 * dd + v_chunk), b);
                        if (tail) {
                            b[0] &= keep0;
                            b[1] &= keep1;
                            b[2] &= keep0;
                            b[3] &= keep1;
                        }
                        mma_16816(o[2 * dd], pf[s], b[0], b[1]);
                        mma_16816(o[2 * dd + 1], pf[s], b[2], b[3]);
                        mma_16816(o[2 * dd], rest[s], b[0], b[1]);
                        mma_16816(o[2 * dd + 1], rest[s], b[2], b[3]);
                    }
                }
            }
            // The last tile's slot is kept for the merge below.
            if (i + 1 < item.count) {
                __syncwarp();
                if (lane == 0) mbar_arrive(empty(slot));
            }
        }

        // ---- the key groups' results become one, in the slot of the last tile ----
        const int last_slot = (it - 1) % C::kStages;
        float* merge = reinterpret_cast<float*>(smem + last_slot * C::kStage);
        // [key group][row][column], the columns of a row exchanged in groups of 8 so that the rows of a half
        // warp fall on different banks.
        auto merge_at = [&](int which, int row, int column) -> float2* {
            return reinterpret_cast<float2*>(merge + (which * 16 * MT + row) * D + (column ^ ((row & 3) * 8)));
        };
        float* row_stats = stats + 16 * mt + g;         // [key group][row]: maxima, then sums
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, d);
            l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        if (t == 0) {
            row_stats[kg * 16 * MT] = m0;
            row_stats[kg * 16 * MT + 8] = m1;
            row_stats[C::kStats + kg * 16 * MT] = l0;
            row_stats[C::kStats + kg * 16 * MT + 8] = l1;
        }
        named_barrier(1, kNarrowWarps * 32);        // all warps are done with the slot's tile
        // Weight of key group `which` of a row, whose largest maximum is `all`.
        auto weight = [&](const float* at, int which, float all) {
            const float mw = at[which * 16 * MT];
            return mw == -INFINITY ? 0.0f : ex2_approx((mw - all) * sl2);
        };
        auto largest = [&](const float* at) {
            float all = at[0];
#pragma unroll
            for (int w = 1; w < kGroups; ++w) all = fmaxf(all, at[w * 16 * MT]);
            return all;
        };
        if (busy) {
            const float w0 = weight(row_stats, kg, largest(row_stats)), w1 = weight(row_stats + 8, kg, largest(row_stats + 8));
#pragma unroll
            for (int j = 0; j < kNTiles; ++j) {
                *merge_at(kg, 16 * mt + g, 8 * j + 2 * t) = make_float2(o[j][0] * w0, o[j][1] * w0);
                if (rows > 16 * mt + 8)
                    *merge_at(kg, 16 * mt + g + 8, 8 * j + 2 * t) = make_float2(o[j][2] * w1, o[j][3] * w1);
            }
        }
        named_barrier(1, kNarrowWarps * 32);
        // Warp w adds up and writes columns [w * D / 4, (w + 1) * D / 4) of every row.
        float* part = p.partial + static_cast<long long>(item.part) * C::kPartFloats;
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e) {
            const int row = 8 * e + g;
            if (!ok || row >= rows) continue;
            const float* at = stats + row;
            const float all = largest(at);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kGroups; ++w) sum += weight(at, w, all) * at[C::kStats + w * 16 * MT];
            const int tok = row / group;
            __nv_bfloat16* out = p.o + static_cast<long long>(item.token0 + tok) * p.o_token +
                                 static_cast<long long>(item.head0 + row - tok * group) * p.o_head;
            const float inv = 1.0f / sum;
#pragma unroll
            for (int j = 0; j < kNTiles / 4; ++j) {
                const int column = warp * (D / 4) + 8 * j + 2 * t;
                float2 a = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kGroups; ++w) {
                    const float2 v = *merge_at(w, row, column);
                    a.x += v.x;
                    a.y += v.y;
                }
                if (item.part < 0) *reinterpret_cast<uint32_t*>(out + column) = pack_bf16x2(a.x * inv, a.y * inv);
                else *reinterpret_cast<float2*>(part + row * D + column) = a;
            }
            if (item.part >= 0 && warp == 0 && t == 0) {
                part[16 * MT * D + row] = all;
                part[16 * MT * D + 16 * MT + row] = sum;
            }
        }
        // The slot goes back to the copies: what was read and written here comes before them.
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(last_slot));
    }
}

// =============================================================================
// Wide kernel: requests of more query rows per K/V head than the narrow kernel takes (chunks of tokens)
// =============================================================================
// The query rows of a K/V head (token * group + head in group) are taken 128 at a time as the M
// of tcgen05 products, so that all heads of a group share each K/V tile; a block is two such
// tiles (256 rows) that ping-pong between two softmax warpgroups, as in the dense kernel. The
// arithmetic is 4 D operations per (row, key) against 4 D bytes per key and block, so the tensor
// pipe and the exponentials bound it, not memory. The work of all requests, K/V heads and blocks
// is one line of 128-key tiles (request, head, block, key; each block preceded by kWideGap idle units
// that stand for its set-up and epilogue) of which each of the grid's CTAs (one per SM, persistent)
// takes an equal stretch; blocks that cross a border are merged from parts. Within a CTA the K/V ring
// runs on across blocks, and the first products of a block overlap the epilogue of the one before.
//
// Warps: 0-3 and 4-7 softmax, O correction and epilogue of Q tile 0 and 1 (one thread per row);
// 8 MMA issuer; 9 and 10 TMA producers of Q and K and of V; 11 walks the line, hands out the segments,
// and zeroes what V's last page holds behind the last key (a weight of zero does not silence a NaN).
// The lazily moved exponent base is that of the dense kernel (fa_sm100.cu); tensor memory is not. A softmax
// warpgroup reads its whole S into registers at once, so S is free long before P is written. P has columns of its
// own here, and Q K^T of the next key tile runs during the softmax of this one: at D = 64 each Q tile has its
// S, at D = 128, where S, P and O of two tiles would not fit, the two take turns with one. What bounds the kernel now is
// the softmax: about 3400 cycles per key tile of a block of two Q tiles, of which the special-function
// unit needs 2048 (a part of the exponentials as cubics on the FMA pipe was slower: 403 us against 394). P is rounded to
// bf16 for the product with V, as in the dense kernel: a second product for the rest would cost the tensor
// pipe a third more, and at D = 128 tensor memory has no room for it. The result is off by 0.0024 of its size,
// against 0.0017 where it alone is rounded. Measured (B200, 32/8 heads, D = 128): 2048 new tokens behind 14336 cached
// 385 to 400 us in short runs, up to 1340 TFLOP/s (457 us a call in long ones, at the power limit), with S and P in
// the same columns 405; a causal prompt of 8192 tokens 435 us (455); 16
// requests of 16 new tokens (64 rows) behind up to 8192 71 us, 4.3 TB/s.
constexpr int kWideThreads = 384;
constexpr int kWideMinUnits = 4;        // units a CTA takes at least, more than a tile's (256 new tokens: 17.8 us; 2: 19.4, 8: 20.7)
// 216 / 72 registers made the MMA issuer spill, and a load by it waits for its queued MMAs: 493 us against 462 (chunk
// of 2048 tokens).
constexpr uint32_t kWideRegsLaunch = 168, kWideRegsSoftmax = 200, kWideRegsOther = 104;
static_assert(2 * 128 * kWideRegsSoftmax + 128 * kWideRegsOther <= kWideThreads * kWideRegsLaunch,
              "the warpgroup register split must fit in the registers the CTA launches with");

enum WideSite : uint32_t {
    kSiteWideSched = 40, kSiteWideQ = 41, kSiteWideK = 42, kSiteWideV = 43, kSiteWideP = 44, kSiteWideEmpty = 45,
    kSiteWideS = 46, kSiteWideO = 47, kSiteWideTail = 48,
};

template <int D>
struct WideCfg {
    static constexpr int kSub = D / 64;                         // 64-column swizzle blocks per row
    static constexpr int kSubBytes = kWideRows * 128;
    static constexpr int kTileBytes = kSub * kSubBytes;         // one Q, K or V tile
    static constexpr int kStages = D == 128 ? 4 : 8;
    static constexpr int kRingOff = 2 * kTileBytes;
    static constexpr int kBarOff = kRingOff + kStages * kTileBytes;
    static constexpr int kBarQFull = 0, kBarQEmpty = 1;
    static constexpr int kBarKvFull = 2, kBarKvEmpty = 2 + kStages;
    // Per Q tile, each completed once per key tile: S computed, S read (by a lane of each warp), half of P written,
    // P written, the product of that half with V done, the whole product done.
    static constexpr int kBarSFull = 2 + 2 * kStages;
    static constexpr int kBarSRead = kBarSFull + 2;
    static constexpr int kBarPHalf = kBarSRead + 2;
    static constexpr int kBarPFull = kBarPHalf + 2;
    static constexpr int kBarPvHalf = kBarPFull + 2;
    static constexpr int kBarPvFull = kBarPvHalf + 2;
    static constexpr int kBarTail = kBarPvFull + 2;              // per ring slot: a V tile to be zeroed in part has landed
    static constexpr int kBarDrain = kBarTail + kStages;
    static constexpr int kBarSchedFull = kBarDrain + 1;
    static constexpr int kBarSchedEmpty = kBarSchedFull + 2;
    static constexpr int kNumBars = kBarSchedEmpty + 2;
    static constexpr int kMiscOff = kBarOff + kNumBars * 8;     // tensor memory base, abort flag
    static constexpr int kSegOff = (kMiscOff + 8 + 15) / 16 * 16;
    // Epilogue staging per softmax warp: 32 rows of 32 columns, 16 bytes apart so that rows fall on different banks.
    static constexpr int kStageStride = 80;
    static constexpr int kStageOff = kSegOff + 2 * 64;
    static constexpr int kSmemBytes = kStageOff + 8 * 32 * kStageStride + 1024;
    static constexpr bool kOwnS = D == 64;                      // S of Q tile 1 in columns of its own
    static constexpr uint32_t kColS0 = 0, kColS1 = D == 64 ? 384 : 0, kColP0 = 128, kColP1 = 192, kColO0 = 256, kColO1 = 256 + D;
    static constexpr uint32_t kIdescQK = make_idesc_bf16(kWideRows, kWideKeys, false);
    static constexpr uint32_t kIdescPV = make_idesc_bf16(kWideRows, D, true);
    // A part: per Q tile O as [D / 4][128 rows] of float4, then 128 maxima and 128 sums.
    static constexpr int kPartTileFloats = kWideRows * (D + 2);
    static_assert(kSmemBytes <= 232448, "shared memory budget");
};

// A stretch of one block inside a CTA's range.
struct WideSegment {
    int b, h;
    int token0;             // packed row of the block's first token
    int tokens;             // tokens of the block, at most 2 * tokens_per_tile
    int pos0;               // position of its first token
    int kv;                 // keys of the request
    int tile, count;        // key tiles [tile, tile + count) of the block; count 0 ends the walk
    int part;               // place of its part, -1: the whole block, written directly
    int zero_from, zero_to; // rows of the last V tile that must read as zero ([0, 0): none)
    int reserved;
    long long last;         // end of the block's units on the line
    int parts;              // CTAs that share the block
    int reserved2;
};
static_assert(sizeof(WideSegment) == 64, "segment slots");

// For one warp, all lanes with the same arguments.
__device__ inline WideSegment wide_segment(const FaPagedPlan& plan, const RequestFinder& finder, long long x, long long end,
                                           long long share)
{
    WideSegment s;
    const Request r = finder.find(quotient(x, plan.kv_heads));
    s.b = r.b;
    s.h = static_cast<int>(quotient(x - r.start * plan.kv_heads, r.units));
    const long long head_first = r.start * plan.kv_heads + s.h * r.units;
    const int n = r.tokens;
    s.kv = r.kv;
    const int cached = s.kv - n;
    const int span = 2 * tokens_per_tile(plan.heads / plan.kv_heads);
    const bool causal = plan.causal != 0;
    const int lane = threadIdx.x % 32, whole = n / span;
    int lo = 0, blocks = (n - 1) / span + 1;    // the last block in [lo, lo + blocks) whose units begin at or before x
    while (blocks > 1) {
        const int step = (blocks + 31) / 32;
        const bool below = lane * step < blocks &&
                           head_first + wide_units_through(lo + lane * step, whole, span, cached, n, causal) <= x;
        const int at = RequestFinder::last_of(below);
        lo += at * step;
        blocks = min(step, blocks - at * step);
    }
    // The block's tiles lie at first, first + weight, ... of the line; a CTA takes those that begin in its range.
    const long long first = head_first + wide_units_through(lo, whole, span, cached, n, causal) + kWideGap;
    const int weight = wide_weight(lo, span, n);
    const int tiles = static_cast<int>(wide_tiles_of(lo, span, cached, n, causal));
    s.last = first + static_cast<long long>(weight) * tiles;
    if (s.last <= x || s.last > head_first + r.units || !request_in_range(plan, r)) {
        if (lane == 0) record_other_plan();
        s.count = 0;
        s.last = end;
        return s;
    }
    s.token0 = r.token0 + lo * span;
    s.tokens = min(span, n - lo * span);
    s.pos0 = cached + lo * span;
    s.tile = x <= first ? 0 : static_cast<int>((x - first + weight - 1) >> (weight - 1));
    const int stop = end >= s.last ? tiles : end <= first ? 0 : static_cast<int>((end - first + weight - 1) >> (weight - 1));
    s.count = stop - s.tile;        // 0 or less: no tile of the block begins in the rest of the range
    // A block whose first tile is another CTA's leaves its part in the CTA's first place, one whose last tile is
    // another's in the second.
    s.part = s.tile > 0 ? 0 : stop < tiles ? 1 : -1;
    s.parts = static_cast<int>(quotient(first + static_cast<long long>(weight) * (tiles - 1), share) - quotient(first, share)) + 1;
    s.reserved = s.reserved2 = 0;
    // Behind the last key: rows of the last page (pages behind it are zero-filled by the copy).
    const int v0 = (s.tile + s.count - 1) * kWideKeys;
    const int held = (s.kv + plan.page_size - 1) & ~(plan.page_size - 1);
    s.zero_from = s.kv - v0;
    s.zero_to = min(kWideKeys, held - v0);
    if (s.zero_from >= s.zero_to) s.zero_from = s.zero_to = 0;
    return s;
}

__device__ __forceinline__ long long wide_share(long long total, int ctas)
{
    const long long even = ceil_div(total, ctas);
    return even > kWideMinUnits ? even : kWideMinUnits;
}

// A matrix descriptor (fa_sm100_ptx.cuh) as its low word -- address and leading offset, which a step along
// K adds to -- and its high word, the same for all tiles: only one register changes between MMAs.
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo_bytes) { return (saddr >> 4) | (lbo_bytes >> 4) << 16; }
__device__ __forceinline__ uint64_t desc_of(uint32_t low)
{
    constexpr uint32_t kHigh = (1024u >> 4) | 1u << 14 | 2u << 29;     // 8-row groups 1024 bytes apart, version 1, 128-byte swizzle
    return static_cast<uint64_t>(kHigh) << 32 | low;
}

// The products of one Q tile with one K or V tile, from the low words of the tiles' descriptors.
template <int D>
__device__ __forceinline__ void wide_issue_qk(uint32_t d_tmem, uint32_t q_low, uint32_t k_low)
{
    using C = WideCfg<D>;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = static_cast<uint32_t>(((kk >> 2) * C::kSubBytes + (kk & 3) * 32) >> 4);
        umma_ss(d_tmem, desc_of(q_low + off), desc_of(k_low + off), C::kIdescQK, kk > 0 ? 1u : 0u);
    }
}

template <int D, int kFirst, int kLast>
__device__ __forceinline__ void wide_issue_pv(uint32_t d_tmem, uint32_t p_tmem, uint32_t v_low, bool accumulate)
{
    using C = WideCfg<D>;
#pragma unroll
    for (int kk = kFirst; kk < kLast; ++kk)
        umma_ts(d_tmem, p_tmem + static_cast<uint32_t>(kk * 8), desc_of(v_low + static_cast<uint32_t>((kk * 16 * 128) >> 4)),
                C::kIdescPV, (accumulate || kk > 0) ? 1u : 0u);
}

template <int D>
__global__ void __launch_bounds__(kWideThreads, 1)
paged_wide_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedParams p)
{
    using C = WideCfg<D>;
    const FaPagedPlan& plan = p.plan;
    // In this order: the narrow kernel relies on it.
    grid_dependency_wait();
    grid_dependents_launch();
    const long long* start = wide_starts(plan.schedule, plan.num_seqs);
    const long long total = start[plan.num_seqs] * plan.kv_heads;
    const long long share = wide_share(total, gridDim.x);
    const long long begin = share * blockIdx.x;
    // By one thread: work for a narrow kernel that this call has none of.
    auto check_narrow = [&]() {
        if (blockIdx.x == 0 && !p.narrow_follows && narrow_starts(plan.schedule)[plan.num_seqs] != 0) record_other_plan();
    };
    if (begin >= total) {
        if (threadIdx.x == 0) {
            check_narrow();
            p.wide_merges[blockIdx.x] = Merge{};
        }
        return;
    }
    const long long end = begin + share < total ? begin + share : total;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    const uint32_t ring = base + C::kRingOff;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kMiscOff);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + C::kMiscOff + 4);
    WideSegment* segments = reinterpret_cast<WideSegment*>(smem + C::kSegOff);
    auto bar = [&](int index) -> uint32_t { return base + C::kBarOff + static_cast<uint32_t>(index) * 8u; };
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    constexpr int kMma = 8, kLoadK = 9, kLoadV = 10;
    constexpr int kReaders = 11;            // warps that read a segment slot

    if (warp == 0) {
        for (int i = lane; i < C::kNumBars; i += 32) {
            uint32_t count = 1;
            if (i >= C::kBarSRead && i < C::kBarPHalf) count = 4;
            if (i >= C::kBarPHalf && i < C::kBarPvHalf) count = 128;
            if (i >= C::kBarSchedEmpty) count = kReaders;
            mbar_init(bar(i), count);
        }
        if (lane == 0) *abort_flag = 0u;
        fence_mbarrier_init();
    }
    if (warp == kMma) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int group = plan.heads / plan.kv_heads;
    const int per_tile = tokens_per_tile(group);

    // Waits for segment number sg; false: gave up. Once its fields are read, release_segment.
    auto await_segment = [&](int sg) -> bool {
        return __all_sync(0xffffffffu, wait_paged(bar(C::kBarSchedFull + (sg & 1)), (sg >> 1) & 1, abort_flag, kSiteWideSched));
    };
    auto release_segment = [&](int sg) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kBarSchedEmpty + (sg & 1)));
    };

    if (warp >= kMma) {
        regs_decrease<kWideRegsOther>();
        if (warp == kLoadK || warp == kLoadV) {
            // ======================= TMA producers =============================
            // One warp copies Q and K, one V: pages of 16 tokens make 32 boxes of a key tile, more than one warp
            // can issue in the time of a tile. Ring slots alternate between K and V.
            const int is_v = warp == kLoadV ? 1 : 0;
            const void* map = is_v ? static_cast<const void*>(&tm_v) : static_cast<const void*>(&tm_k);
            const int rows = plan.page_size < kWideKeys ? plan.page_size : kWideKeys;
            const int pages = kWideKeys / rows;
            const bool active = lane < pages * C::kSub;
            const int page_of_tile = lane / C::kSub, block = lane % C::kSub;
            const uint32_t offset = static_cast<uint32_t>(block * C::kSubBytes + page_of_tile * rows * 128);
            int ri = is_v;              // ring index of the next tile
            int q_loads = 0;
            uint32_t tail_slots = 0, tail_parity = 0;      // slots whose latest load went by the tail barrier; their phases
            bool ok = true;
            for (int sg = 0; ok; ++sg) {
                ok = await_segment(sg);
                if (!ok) break;
                const WideSegment& seg = segments[sg & 1];
                const int count = seg.count, first_tile = seg.tile, head = seg.h, token0 = seg.token0;
                const int tiles = seg.tokens > per_tile ? 2 : 1;
                const bool has_tail = seg.zero_to > seg.zero_from;
                const int held = (seg.kv + plan.page_size - 1) >> p.page_shift;
                const int* table = plan.block_table + static_cast<long long>(seg.b) * plan.table_stride;
                release_segment(sg);
                if (count == 0) break;
                if (!is_v) {
                    if (sg > 0 && !__all_sync(0xffffffffu, wait_paged(bar(C::kBarQEmpty), (sg - 1) & 1, abort_flag, kSiteWideQ))) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar(C::kBarQFull), static_cast<uint32_t>(tiles * C::kSub * 128 * group * per_tile));
                        for (int t = 0; t < tiles; ++t)
                            for (int sub = 0; sub < C::kSub; ++sub)
                                tma_load_3d(base + t * C::kTileBytes + sub * C::kSubBytes, &tm_q, bar(C::kBarQFull), sub * 64,
                                            head * group, token0 + t * per_tile);
                    }
                    ++q_loads;
                }
                auto page_at = [&](int tile) -> int {
                    // num_pages is out of the map's range: such a box reads as zeros.
                    const int i = ((tile * kWideKeys) >> p.page_shift) + page_of_tile;
                    if (!active || i >= held) return plan.num_pages;
                    const int page = table[i];     // an ordinary load, as in the narrow kernel
                    if (page >= 0 && page < plan.num_pages) return page;
                    atomicOr(&g_paged_error_word, FA_ERROR_BAD_PAGE);
                    return plan.num_pages;
                };
                int page = page_at(first_tile);
                for (int i = 0; i < count; ++i, ri += 2) {
                    const int row = pages > 1 ? 0 : ((first_tile + i) * kWideKeys) & (plan.page_size - 1);
                    const int slot = ri % C::kStages, use = ri / C::kStages;
                    if (use > 0 && !__all_sync(0xffffffffu, wait_paged(bar(C::kBarKvEmpty + slot), (use - 1) & 1, abort_flag,
                                                                       kSiteWideEmpty))) {
                        ok = false;
                        break;
                    }
                    // A V tile to be zeroed in part lands on the tail barrier; warp 11 then completes the slot's.
                    const bool tail = is_v && i + 1 == count && has_tail;
                    const uint32_t landed = bar((tail ? C::kBarTail : C::kBarKvFull) + slot);
                    tail_slots = tail ? tail_slots | (1u << slot) : tail_slots & ~(1u << slot);
                    if (tail) tail_parity ^= 1u << slot;
                    if (lane == 0) mbar_arrive_expect_tx(landed, C::kTileBytes);
                    __syncwarp();
                    if (active)
                        tma_load_4d(ring + slot * C::kTileBytes + offset, map, landed, block * 64, row, head, page);
                    if (i + 1 < count) page = page_at(first_tile + i + 1);
                }
            }
            if (!ok && lane == 0) {
                if (q_loads > 0) drain_paged(bar(C::kBarQFull), (q_loads - 1) & 1);
                for (int i = ri > C::kStages ? ri - C::kStages : is_v; i < ri; i += 2) {
                    const int slot = i % C::kStages;
                    if (tail_slots >> slot & 1u) drain_paged(bar(C::kBarTail + slot), (tail_parity >> slot & 1u) ^ 1u);
                    else drain_paged(bar(C::kBarKvFull + slot), (i / C::kStages) & 1);
                }
            }
        } else if (warp == kMma) {
            // ======================= MMA issuer ================================
            // Anything but MMAs that this thread does waits until the MMAs it has queued are done, so all it
            // needs is in registers before a segment's loop.
            const uint32_t t_s = tmem_base + C::kColS0, t_s1 = tmem_base + C::kColS1, t_p0 = tmem_base + C::kColP0, t_p1 = tmem_base + C::kColP1;
            const uint32_t t_o0 = tmem_base + C::kColO0, t_o1 = tmem_base + C::kColO1;
            const uint32_t q0 = desc_low(base, 16), q1 = desc_low(base + C::kTileBytes, 16);
            const uint32_t k_ring = desc_low(ring, 16), v_ring = desc_low(ring, C::kSubBytes);
            auto in_slot = [](uint32_t low, int i) { return low + static_cast<uint32_t>(i % C::kStages) * (C::kTileBytes >> 4); };
            auto empty_bar = [&](int i) -> uint32_t { return bar(C::kBarKvEmpty + i % C::kStages); };
            int ri = 0;                         // ring index of the segment's first K tile
            uint32_t par0 = 0, par1 = 0;        // parities of the Q tiles' barriers
            bool ok = true;
            auto wait = [&](int index, uint32_t parity, uint32_t site) { return wait_paged(bar(index), parity, abort_flag, site); };
            auto wait_ring = [&](int i, uint32_t site) {
                return wait_paged(bar(C::kBarKvFull + i % C::kStages), (i / C::kStages) & 1, abort_flag, site);
            };
            // The products of a segment of one Q tile: Q K^T of the next key tile is issued once S of this one is read.
            auto issue_one = [&](int count) -> bool {
                wide_issue_qk<D>(t_s, q0, in_slot(k_ring, ri));
                umma_commit(bar(C::kBarSFull + 0));
                umma_commit(empty_bar(ri));
                if (count == 1) umma_commit(bar(C::kBarQEmpty));
                for (int j = 0; j < count; ++j) {
                    const int vi = ri + 2 * j + 1, ki = vi + 1;
                    if (j + 1 < count) {
                        if (!wait_ring(ki, kSiteWideK)) return false;
                        if (!wait(C::kBarSRead + 0, par0, kSiteWideP)) return false;
                        tc_fence_after();
                        wide_issue_qk<D>(t_s, q0, in_slot(k_ring, ki));
                        umma_commit(bar(C::kBarSFull + 0));
                        umma_commit(empty_bar(ki));
                        if (j + 2 == count) umma_commit(bar(C::kBarQEmpty));
                    }
                    if (!wait_ring(vi, kSiteWideV)) return false;
                    if (!wait(C::kBarPHalf + 0, par0, kSiteWideP)) return false;
                    tc_fence_after();
                    wide_issue_pv<D, 0, 4>(t_o0, t_p0, in_slot(v_ring, vi), j > 0);
                    umma_commit(bar(C::kBarPvHalf + 0));
                    if (!wait(C::kBarPFull + 0, par0, kSiteWideP)) return false;
                    tc_fence_after();
                    wide_issue_pv<D, 4, 8>(t_o0, t_p0, in_slot(v_ring, vi), true);
                    umma_commit(bar(C::kBarPvFull + 0));
                    umma_commit(empty_bar(vi));
                    par0 ^= 1u;
                }
                return true;
            };
            // The products of a segment of two Q tiles. Where they take turns with S, tile 1's Q K^T follows when tile 0
            // has read its S, tile 0's of the next key tile when tile 1 has.
            auto issue_two = [&](int count) -> bool {
                wide_issue_qk<D>(t_s, q0, in_slot(k_ring, ri));
                umma_commit(bar(C::kBarSFull + 0));
                if (!C::kOwnS && !wait(C::kBarSRead + 0, par0, kSiteWideP)) return false;
                tc_fence_after();
                wide_issue_qk<D>(t_s1, q1, in_slot(k_ring, ri));
                umma_commit(bar(C::kBarSFull + 1));
                umma_commit(empty_bar(ri));
                if (count == 1) umma_commit(bar(C::kBarQEmpty));
                for (int j = 0; j < count; ++j) {
                    const int vi = ri + 2 * j + 1, ki = vi + 1;
                    const bool more = j + 1 < count;
                    if (more) {
                        if (!wait_ring(ki, kSiteWideK)) return false;
                        if (!wait(C::kBarSRead + (C::kOwnS ? 0 : 1), C::kOwnS ? par0 : par1, kSiteWideP)) return false;
                        tc_fence_after();
                        wide_issue_qk<D>(t_s, q0, in_slot(k_ring, ki));
                        umma_commit(bar(C::kBarSFull + 0));
                    }
                    if (!wait_ring(vi, kSiteWideV)) return false;
                    if (!wait(C::kBarPHalf + 0, par0, kSiteWideP)) return false;
                    tc_fence_after();
                    wide_issue_pv<D, 0, 4>(t_o0, t_p0, in_slot(v_ring, vi), j > 0);
                    umma_commit(bar(C::kBarPvHalf + 0));
                    if (!wait(C::kBarPFull + 0, par0, kSiteWideP)) return false;
                    tc_fence_after();
                    wide_issue_pv<D, 4, 8>(t_o0, t_p0, in_slot(v_ring, vi), true);
                    umma_commit(bar(C::kBarPvFull + 0));
                    par0 ^= 1u;
                    if (more) {
                        if (!wait(C::kBarSRead + (C::kOwnS ? 1 : 0), C::kOwnS ? par1 : par0, kSiteWideP)) return false;
                        tc_fence_after();
                        wide_issue_qk<D>(t_s1, q1, in_slot(k_ring, ki));
                        umma_commit(bar(C::kBarSFull + 1));
                        umma_commit(empty_bar(ki));
                        if (j + 2 == count) umma_commit(bar(C::kBarQEmpty));    // the segment's last S is on its way
                    }
                    if (!wait(C::kBarPHalf + 1, par1, kSiteWideP)) return false;
                    tc_fence_after();
                    wide_issue_pv<D, 0, 4>(t_o1, t_p1, in_slot(v_ring, vi), j > 0);
                    umma_commit(bar(C::kBarPvHalf + 1));
                    if (!wait(C::kBarPFull + 1, par1, kSiteWideP)) return false;
                    tc_fence_after();
                    wide_issue_pv<D, 4, 8>(t_o1, t_p1, in_slot(v_ring, vi), true);
                    umma_commit(bar(C::kBarPvFull + 1));
                    umma_commit(empty_bar(vi));
                    par1 ^= 1u;
                }
                return true;
            };
            for (int sg = 0; ok; ++sg) {
                ok = await_segment(sg);
                if (!ok) break;
                const int count = segments[sg & 1].count;
                const bool two = segments[sg & 1].tokens > per_tile;
                release_segment(sg);
                if (count == 0) break;
                if (elect_one()) {
                    ok = wait(C::kBarQFull, sg & 1, kSiteWideQ) && wait_ring(ri, kSiteWideK);
                    if (ok) {
                        tc_fence_after();
                        ok = two ? issue_two(count) : issue_one(count);
                        ri += 2 * count;
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
            }
            if (elect_one()) {
                // Every MMA issued above must finish before tensor memory is released.
                umma_commit(bar(C::kBarDrain));
                drain_paged(bar(C::kBarDrain), 0);
            }
            __syncwarp();
        } else {
            // ======================= the walk along the line, and V behind the last key
            const RequestFinder finder(plan, start);
            long long x = begin;
            Merge merge{};
            int ri = 0;                                     // ring index behind the segment before
            int zero_from = 0, zero_to = 0, zero_slot = 0;  // of the segment before
            uint32_t parity = 0;
            const bool go = p.inject_stall == 0 ||
                            __all_sync(0xffffffffu, wait_paged(bar(C::kBarSchedEmpty), 0, abort_flag, kSiteWideSched));
            for (int sg = 0; go; ++sg) {
                if (sg > 1 && !__all_sync(0xffffffffu, wait_paged(bar(C::kBarSchedEmpty + (sg & 1)), ((sg >> 1) - 1) & 1,
                                                                  abort_flag, kSiteWideSched)))
                    break;
                WideSegment s;
                s.count = 0;
                while (x < end && s.count <= 0) {
                    s = wide_segment(plan, finder, x, end, share);
                    x = s.last;
                    if (s.count < 0) s.count = 0;
                }
                if (s.count > 0) {
                    if (s.part == 1) merge = {s.parts, s.token0, s.tokens, s.h * group};
                    if (s.part >= 0) s.part += 2 * static_cast<int>(blockIdx.x);
                }
                if (lane == 0) {
                    segments[sg & 1] = s;
                    mbar_arrive(bar(C::kBarSchedFull + (sg & 1)));
                }
                // The segment before: the rows behind the last key of its last V tile.
                if (zero_from < zero_to) {
                    if (!__all_sync(0xffffffffu, wait_paged(bar(C::kBarTail + zero_slot), parity >> zero_slot & 1u, abort_flag,
                                                            kSiteWideTail)))
                        break;
                    parity ^= 1u << zero_slot;
                    const int bytes = (zero_to - zero_from) * 128;
                    for (int sub = 0; sub < C::kSub; ++sub) {
                        uint8_t* at = smem + C::kRingOff + zero_slot * C::kTileBytes + sub * C::kSubBytes + zero_from * 128;
                        for (int i = lane * 16; i < bytes; i += 512) *reinterpret_cast<uint4*>(at + i) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(C::kBarKvFull + zero_slot));
                }
                if (s.count == 0) break;
                ri += 2 * s.count;
                zero_from = s.zero_from;
                zero_to = s.zero_to;
                zero_slot = (ri - 1) % C::kStages;
            }
            if (lane == 0) {
                p.wide_merges[blockIdx.x] = merge;
                check_narrow();
            }
        }
        __syncwarp();
    } else {
        // ======================= softmax / correction / epilogue ================
        regs_increase<kWideRegsSoftmax>();
        const int t = warp / 4;                    // Q tile of this warpgroup
        const int quarter = warp % 4;
        const int r = quarter * 32 + lane;         // row within the Q tile == tensor-memory lane
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t t_s = lane_base + (t == 0 ? C::kColS0 : C::kColS1);
        const uint32_t t_p = lane_base + (t == 0 ? C::kColP0 : C::kColP1);
        const uint32_t t_o = lane_base + (t == 0 ? C::kColO0 : C::kColO1);
        const int tok = t * per_tile + r / group;       // token of this row within its block
        const float sl2 = p.scale_log2;
        const uint64_t c2 = f2_pack(sl2, sl2);
        uint32_t phase = 0;     // parity of this Q tile's barriers

        auto rescale_o = [&](float scale) {
            const uint64_t a2 = f2_pack(scale, scale);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(t_o + static_cast<uint32_t>(c * 32), o);
                tmem_wait_ld();
                reg_fence32(o);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float o0, o1;
                    f2_unpack(fmul2(f2_pack(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), a2), o0, o1);
                    o[2 * i] = __float_as_uint(o0);
                    o[2 * i + 1] = __float_as_uint(o1);
                }
                tmem_st32(t_o + static_cast<uint32_t>(c * 32), o);
            }
        };
        // 64 scores on base `mb`: P as bf16 pairs, the 32-bit sum and the raw maximum.
        auto exp_half = [&](const uint32_t (&lo)[32], const uint32_t (&hi)[32], float mb, float& half_sum, float& half_max,
                            uint32_t p_tmem) {
            const uint64_t nb2 = f2_pack(-mb, -mb);
            uint64_t sum_a = f2_pack(0.0f, 0.0f), sum_b = f2_pack(0.0f, 0.0f);
            float ma = fmaxf(__uint_as_float(lo[0]), __uint_as_float(lo[1])), mb_ = __uint_as_float(hi[0]);
            uint32_t out[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t (&src)[32] = (i < 16) ? lo : hi;
                const int k = (i & 15) * 2;
                if (i >= 16) mb_ = max3f(mb_, __uint_as_float(src[k]), __uint_as_float(src[k + 1]));
                else if (i > 0) ma = max3f(ma, __uint_as_float(src[k]), __uint_as_float(src[k + 1]));
                const uint64_t x = ffma2(f2_pack(__uint_as_float(src[k]), __uint_as_float(src[k + 1])), c2, nb2);
                float x0, x1;
                f2_unpack(x, x0, x1);
                const uint64_t pr = f2_pack(ex2_approx(x0), ex2_approx(x1));
                if (i & 1) sum_b = fadd2(sum_b, pr);
                else sum_a = fadd2(sum_a, pr);
                float p0, p1;
                f2_unpack(pr, p0, p1);
                out[i] = pack_bf16x2(p0, p1);
                if (i == 15) tmem_st16(p_tmem, *reinterpret_cast<uint32_t (*)[16]>(&out[0]));
                if (i == 31) tmem_st16(p_tmem + 16, *reinterpret_cast<uint32_t (*)[16]>(&out[16]));
            }
            float sa0, sa1, sb0, sb1;
            f2_unpack(sum_a, sa0, sa1);
            f2_unpack(sum_b, sb0, sb1);
            half_sum = (sa0 + sa1) + (sb0 + sb1);
            half_max = fmaxf(ma, mb_);
        };

        bool ok = true;
        for (int sg = 0; ok; ++sg) {
            // The slot stays this segment's until the epilogue has read it.
            ok = await_segment(sg);
            if (!ok) break;
            const WideSegment& seg = segments[sg & 1];
            const int count = seg.count;
            if (count == 0) break;
            const bool one = seg.tokens <= per_tile;    // this block has one Q tile
            if (t == 1 && one) {
                release_segment(sg);
                continue;
            }
            const int tile = seg.tile;
            const int limit = plan.causal ? min(seg.pos0 + tok, seg.kv - 1) : seg.kv - 1;
            // First key tile of the stretch that some row of this Q tile must not see all of.
            const int mask_from = (plan.causal ? seg.pos0 + t * per_tile + 1 : seg.kv) / kWideKeys - tile;
            float row_max = -INFINITY, row_sum = 0.0f, m_base = 0.0f;
            for (int j = 0; j < count; ++j, phase ^= 1u) {
                ok = __all_sync(0xffffffffu, wait_paged(bar(C::kBarSFull + t), phase, abort_flag, kSiteWideS));
                if (!ok) break;
                tc_fence_after();
                uint32_t sc[4][32];
                tmem_ld32(t_s + 0, sc[0]);
                tmem_ld32(t_s + 32, sc[1]);
                tmem_ld32(t_s + 64, sc[2]);
                tmem_ld32(t_s + 96, sc[3]);
                tmem_wait_ld();
                reg_fence32(sc[0]);
                reg_fence32(sc[1]);
                reg_fence32(sc[2]);
                reg_fence32(sc[3]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(C::kBarSRead + t));
                const int key0 = (tile + j) * kWideKeys;
                if (j >= mask_from && __any_sync(0xffffffffu, limit < key0 + kWideKeys - 1)) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (key0 + c * 32 + i > limit) sc[c][i] = __float_as_uint(-INFINITY);
                }
                if (j == 0) {
                    float mx[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float a = __uint_as_float(sc[c][0]), b = __uint_as_float(sc[c][1]);
#pragma unroll
                        for (int i = 2; i < 32; i += 2) {
                            a = fmaxf(a, __uint_as_float(sc[c][i]));
                            b = fmaxf(b, __uint_as_float(sc[c][i + 1]));
                        }
                        mx[c] = fmaxf(a, b);
                    }
                    row_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    m_base = row_max == -INFINITY ? 0.0f : row_max * sl2;
                }
                if (j > 0) {
                    // O and P are the previous tile's until its product with V is done.
                    ok = __all_sync(0xffffffffu, wait_paged(bar(C::kBarPvFull + t), phase ^ 1u, abort_flag, kSiteWideO));
                    if (!ok) break;
                    tc_fence_after();
                }
                float o_scale = 1.0f;       // O correction owed before the first PV of this tile reads O
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float hsum, hmax;
                    exp_half(sc[2 * h], sc[2 * h + 1], m_base, hsum, hmax, t_p + static_cast<uint32_t>(32 * h));
                    const bool need = (hmax - row_max) * sl2 > kRebase;
                    if (__any_sync(0xffffffffu, need)) {
                        const float m_new = need ? hmax : row_max;
                        const float alpha = need ? ex2_approx(row_max * sl2 - m_new * sl2) : 1.0f;
                        row_sum *= alpha;
                        row_max = m_new;
                        m_base = row_max == -INFINITY ? 0.0f : row_max * sl2;
                        if (h == 0) {
                            o_scale = alpha;
                        } else {
                            // The first-half PV of this tile may be running on the old base: let it finish, then
                            // correct O, its contribution included.
                            ok = __all_sync(0xffffffffu, wait_paged(bar(C::kBarPvHalf + t), phase, abort_flag, kSiteWideO));
                            if (!ok) break;
                            tc_fence_after();
                            rescale_o(alpha);
                        }
                        exp_half(sc[2 * h], sc[2 * h + 1], m_base, hsum, hmax, t_p + static_cast<uint32_t>(32 * h));
                    }
                    row_sum += hsum;
                    if (h == 0 && j > 0 && __any_sync(0xffffffffu, o_scale != 1.0f)) rescale_o(o_scale);
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(bar((h == 0 ? C::kBarPHalf : C::kBarPFull) + t));
                }
                if (!ok) break;
            }
            if (!ok) break;

            // ---- epilogue: O from tensor memory, to its rows or to this stretch's part ----
            ok = __all_sync(0xffffffffu, wait_paged(bar(C::kBarPvFull + t), phase ^ 1u, abort_flag, kSiteWideO));
            if (!ok) break;
            tc_fence_after();
            const int part = seg.part;
            // A row of 32 columns is 64 bytes: staged in shared memory, four lanes write one row, so that a warp's
            // store touches 8 rows and not 32. This lane writes rows 8 i + lane / 4 of the warp's 32.
            __nv_bfloat16* out[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = quarter * 32 + 8 * i + lane / 4;
                const int row_tok = t * per_tile + row / group;
                const bool real = row < per_tile * group && row_tok < seg.tokens;
                out[i] = real ? p.o + static_cast<long long>(seg.token0 + row_tok) * p.o_token +
                                    static_cast<long long>(seg.h * group + row % group) * p.o_head + (lane % 4) * 8
                              : nullptr;
            }
            release_segment(sg);
            if (part < 0) {
                const float inv = 1.0f / row_sum;
                const uint32_t stage = base + C::kStageOff + static_cast<uint32_t>(warp * 32 * C::kStageStride);
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(t_o + static_cast<uint32_t>(c * 32), o);
                    tmem_wait_ld();
                    reg_fence32(o);
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[i] = pack_bf16x2(__uint_as_float(o[8 * q + 2 * i]) * inv, __uint_as_float(o[8 * q + 2 * i + 1]) * inv);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                                     :: "r"(stage + lane * C::kStageStride + q * 16), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                                     : "memory");
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint4 w;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                                     : "r"(stage + (8 * i + lane / 4) * C::kStageStride + (lane % 4) * 16) : "memory");
                        if (out[i] != nullptr) *reinterpret_cast<uint4*>(out[i] + c * 32) = w;
                    }
                }
            } else {
                float* mine = p.wide_partial + (static_cast<long long>(part) * 2 + t) * C::kPartTileFloats;
                float4* columns = reinterpret_cast<float4*>(mine);
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(t_o + static_cast<uint32_t>(c * 32), o);
                    tmem_wait_ld();
                    reg_fence32(o);
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        columns[(c * 8 + q) * kWideRows + r] =
                            make_float4(__uint_as_float(o[4 * q]), __uint_as_float(o[4 * q + 1]),
                                        __uint_as_float(o[4 * q + 2]), __uint_as_float(o[4 * q + 3]));
                }
                mine[D * kWideRows + r] = row_max;
                mine[D * kWideRows + kWideRows + r] = row_sum;
            }
        }
        tc_fence_before();
    }

    __syncthreads();
    if (warp == kMma) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// =============================================================================
// Merging of parts
// =============================================================================
// An item (narrow) or block (wide) that crossed borders between CTAs' ranges left a part in each; they
// are merged in their order, so that a result does not depend on which CTA was done first. A row's
// parts O_i, with maxima m_i and sums l_i, give
//     sum_i w_i O_i / sum_i w_i l_i,   w_i = 2^((m_i - max_i m_i) log2(e) / sqrt(D)).
// What to merge was written down by the CTA with the first part. A few round trips to memory bound
// this, so its blocks are small and launched while the kernel before still runs (programmatic
// dependent launch): about 3 us behind the narrow kernel; behind the wide one, whose parts are 256 rows,
// 5 us for 40 MB of parts at D = 128.
constexpr int kCombineThreads = 128;
constexpr int kCombineColumns = 32;         // wide: columns of a thread

// One row per warp; a lane has D / 32 columns.
template <int D, int MT>
__device__ __forceinline__ void combine_narrow(const PagedParams& p, int cta, int row)
{
    using C = NarrowCfg<D, MT>;
    constexpr int E = D / 32;
    const Merge merge = p.merges[cta];
    const int group = p.plan.heads / p.plan.kv_heads, lane = threadIdx.x % 32;
    if (row >= merge.tokens * group || merge.parts == 0) return;
    const float* first = p.partial + (2LL * cta + 1) * C::kPartFloats;
    auto part = [&](int i) { return i == 0 ? first : first + (2LL * i - 1) * C::kPartFloats; };
    // 32 parts at a time: a lane reads one part's maximum and sum, then all lanes add up its columns.
    float top = -INFINITY, sum = 0.0f, acc[E] = {};
    for (int i0 = 0; i0 < merge.parts; i0 += 32) {
        const int mine = i0 + lane;
        const float m = mine < merge.parts ? part(mine)[16 * MT * D + row] : -INFINITY;
        const float l = mine < merge.parts ? part(mine)[16 * MT * D + 16 * MT + row] : 0.0f;
        float high = fmaxf(m, top);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
        const float keep = top == -INFINITY ? 0.0f : ex2_approx((top - high) * p.scale_log2);
        const float w = m == -INFINITY ? 0.0f : ex2_approx((m - high) * p.scale_log2);
        float wl = w * l;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) wl += __shfl_xor_sync(0xffffffffu, wl, d);
        sum = sum * keep + wl;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= keep;
        top = high;
        const int here = min(32, merge.parts - i0);
#pragma unroll 8
        for (int i = 0; i < here; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            const float* at = part(i0 + i) + row * D + lane * E;
            if constexpr (E == 4) {
                const float4 v = *reinterpret_cast<const float4*>(at);
                acc[0] += wi * v.x;
                acc[1] += wi * v.y;
                acc[2] += wi * v.z;
                acc[3] += wi * v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(at);
                acc[0] += wi * v.x;
                acc[1] += wi * v.y;
            }
        }
    }
    const float inv = 1.0f / sum;
    const int tok = row / group;
    __nv_bfloat16* out = p.o + static_cast<long long>(merge.token0 + tok) * p.o_token +
                         static_cast<long long>(merge.head0 + row - tok * group) * p.o_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2)
        *reinterpret_cast<uint32_t*>(out + e) = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
}

// A block per CTA of the narrow kernel and four rows.
template <int D, int MT>
__global__ void __launch_bounds__(kCombineThreads)
paged_combine_narrow_kernel(const __grid_constant__ PagedParams p)
{
    constexpr int kWarps = kCombineThreads / 32, kRowBlocks = 16 * MT / kWarps;
    const int block = static_cast<int>(blockIdx.x);
    grid_dependents_launch();
    grid_dependency_wait();
    combine_narrow<D, MT>(p, block / kRowBlocks, block % kRowBlocks * kWarps + static_cast<int>(threadIdx.x) / 32);
}

// A block per CTA of the wide kernel, Q tile and group of columns; a thread is a query row.
template <int D>
__global__ void __launch_bounds__(kCombineThreads)
paged_combine_wide_kernel(const __grid_constant__ PagedParams p)
{
    using C = WideCfg<D>;
    constexpr int kGroups = D / kCombineColumns, kQuads = kCombineColumns / 4;
    const int block = static_cast<int>(blockIdx.x), cta = block / (2 * kGroups), t = block / kGroups % 2, c = block % kGroups;
    const int group = p.plan.heads / p.plan.kv_heads, per_tile = tokens_per_tile(group);
    const int r = threadIdx.x, tok = t * per_tile + r / group;
    grid_dependents_launch();
    grid_dependency_wait();
    const Merge merge = p.wide_merges[cta];
    if (merge.parts == 0 || r >= per_tile * group || tok >= merge.tokens) return;
    const float* first = p.wide_partial + ((2LL * cta + 1) * 2 + t) * C::kPartTileFloats;
    auto part = [&](int i) { return i == 0 ? first : first + (2LL * i - 1) * 2 * C::kPartTileFloats; };
    float top = -INFINITY;
#pragma unroll 8
    for (int i = 0; i < merge.parts; ++i) top = fmaxf(top, part(i)[D * kWideRows + r]);
    float4 acc[kQuads] = {};
    float sum = 0.0f;
#pragma unroll 2
    for (int i = 0; i < merge.parts; ++i) {
        const float* at = part(i);
        const float m = at[D * kWideRows + r];
        const float w = m == -INFINITY ? 0.0f : ex2_approx((m - top) * p.scale_log2);
        sum += w * at[D * kWideRows + kWideRows + r];
        const float4* columns = reinterpret_cast<const float4*>(at) + c * kQuads * kWideRows + r;
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            const float4 v = columns[q * kWideRows];
            acc[q].x += w * v.x;
            acc[q].y += w * v.y;
            acc[q].z += w * v.z;
            acc[q].w += w * v.w;
        }
    }
    const float inv = 1.0f / sum;
    __nv_bfloat16* out = p.o + static_cast<long long>(merge.token0 + tok) * p.o_token +
                         static_cast<long long>(merge.head0 + r % group) * p.o_head + c * kCombineColumns;
#pragma unroll
    for (int q = 0; q < kQuads; q += 2)
        *reinterpret_cast<uint4*>(out + q * 4) =
            make_uint4(pack_bf16x2(acc[q].x * inv, acc[q].y * inv), pack_bf16x2(acc[q].z * inv, acc[q].w * inv),
                       pack_bf16x2(acc[q + 1].x * inv, acc[q + 1].y * inv), pack_bf16x2(acc[q + 1].z * inv, acc[q + 1].w * inv));
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
    static std::atomic<int> counts[kMax];       // SM count of each device once known
    cudaError_t err = cudaGetDevice(device);
    if (err != cudaSuccess) return static_cast<int>(err);
    if (*device < 0 || *device >= kMax) return FA_STATUS_INVALID_ARGUMENT;
    if (counts[*device].load() == 0) {
        int major = 0, count = 0;
        err = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *device);
        if (err != cudaSuccess) return static_cast<int>(err);
        if (major != 10) return FA_STATUS_NO_SM100;
        err = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, *device);
        if (err != cudaSuccess) return static_cast<int>(err);
        counts[*device].store(count);
    }
    *sm_count = counts[*device].load();
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
    // The kernels count requests and rows in 32 bits, in steps of up to a block of threads.
    if (plan->num_seqs >= (1 << 30) || plan->total_tokens >= (1 << 30)) return FA_STATUS_INVALID_ARGUMENT;
    // Slots are 32-bit; positions leave room for a tile behind the last key.
    if (static_cast<long long>(plan->num_pages) * plan->page_size > INT_MAX ||
        static_cast<long long>(plan->table_width) * plan->page_size > (1 << 30))
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
        struct { const void* kernel; int bytes; } const narrow[] = {
            {reinterpret_cast<const void*>(paged_narrow_kernel<64, 1>), NarrowCfg<64, 1>::kSmemBytes},
            {reinterpret_cast<const void*>(paged_narrow_kernel<64, 2>), NarrowCfg<64, 2>::kSmemBytes},
            {reinterpret_cast<const void*>(paged_narrow_kernel<128, 1>), NarrowCfg<128, 1>::kSmemBytes},
            {reinterpret_cast<const void*>(paged_narrow_kernel<128, 2>), NarrowCfg<128, 2>::kSmemBytes}};
        cudaError_t err = cudaSuccess;
        for (int i = 0; i < 4 && err == cudaSuccess; ++i)
            err = cudaFuncSetAttribute(narrow[i].kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, narrow[i].bytes);
        const void* const wide[] = {reinterpret_cast<const void*>(paged_wide_kernel<64>),
                                    reinterpret_cast<const void*>(paged_wide_kernel<128>)};
        for (int i = 0; i < 2 && err == cudaSuccess; ++i) {
            err = cudaFuncSetAttribute(wide[i], cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       i == 0 ? WideCfg<64>::kSmemBytes : WideCfg<128>::kSmemBytes);
            // setmaxnreg waits forever for registers that the CTA did not launch with.
            cudaFuncAttributes attributes{};
            if (err == cudaSuccess) err = cudaFuncGetAttributes(&attributes, wide[i]);
            if (err == cudaSuccess && static_cast<uint32_t>(attributes.numRegs) * kWideThreads <
                                          2u * 128u * kWideRegsSoftmax + 128u * kWideRegsOther) {
                state.status = FA_STATUS_BUILD_MISMATCH;
                return;
            }
        }
        state.status = static_cast<int>(err);
    });
    return state.status;
}

// Test only: set by fa_sm100_paged_test_arm_stall for this host thread's next launch.
thread_local bool t_armed_stall = false;

int narrow_ctas(int sms) { return kNarrowCtasPerSm * sms; }

// Workspace: the parts, then the merges, of each kernel.
size_t narrow_parts(int sms, const FaPagedPlan& plan)
{
    return static_cast<size_t>(narrow_ctas(sms)) * 2 * narrow_rows(plan) * (plan.head_dim + 2) * sizeof(float);
}
size_t narrow_workspace(int sms, const FaPagedPlan& plan) { return narrow_parts(sms, plan) + narrow_ctas(sms) * sizeof(Merge); }

size_t wide_parts(int sms, int head_dim)
{
    return static_cast<size_t>(sms) * 2 * 2 * kWideRows * (head_dim + 2) * sizeof(float);
}
size_t wide_workspace(int sms, int head_dim) { return wide_parts(sms, head_dim) + sms * sizeof(Merge); }

// Which kernels a plan's requests can need: decided from the sizes that the host knows.
bool may_be_narrow(const FaPagedPlan& plan) { return plan.heads / plan.kv_heads <= narrow_rows(plan); }
bool may_be_wide(const FaPagedPlan& plan)
{
    return most_rows(plan) > narrow_rows(plan);
}

size_t workspace_bytes_of(const FaPagedPlan& plan, int sms)
{
    return (may_be_narrow(plan) ? narrow_workspace(sms, plan) : 0) +
           (may_be_wide(plan) ? wide_workspace(sms, plan.head_dim) : 0);
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

struct PagedMaps {
    CUtensorMap q;                          // wide
    CUtensorMap wide_k, wide_v;
    CUtensorMap narrow_k, narrow_v;
};

// The wide kernel and the merging of its parts, then the narrow kernel and the merging of its own. The narrow
// kernel needs nothing of the wide one: it fills the SMs that fall idle and runs beside the merging.
template <int D, int MT>
int launch_attention(const PagedMaps& maps, const PagedParams& params, bool wide, bool narrow, int sms, cudaStream_t stream)
{
    int status = FA_STATUS_OK;
    if (wide) {
        status = fa_sm100_internal::launch_early(paged_wide_kernel<D>, sms, kWideThreads, WideCfg<D>::kSmemBytes, stream, maps.q, maps.wide_k,
                        maps.wide_v, params);
        if (status == FA_STATUS_OK)
            status = fa_sm100_internal::launch_early(paged_combine_wide_kernel<D>, sms * 2 * (D / kCombineColumns), kCombineThreads, 0, stream,
                            params);
    }
    if (!narrow || status != FA_STATUS_OK) return status;
    const int ctas = narrow_ctas(sms);
    status = fa_sm100_internal::launch_early(paged_narrow_kernel<D, MT>, ctas, kNarrowThreads, NarrowCfg<D, MT>::kSmemBytes, stream, maps.narrow_k,
                    maps.narrow_v, params);
    if (status != FA_STATUS_OK) return status;
    return fa_sm100_internal::launch_early(paged_combine_narrow_kernel<D, MT>, ctas * (16 * MT / (kCombineThreads / 32)), kCombineThreads, 0, stream,
                  params);
}

}  // namespace

extern "C" {

int fa_sm100_paged_test_arm_stall(void)
{
    t_armed_stall = true;
    return FA_STATUS_OK;
}

size_t fa_sm100_paged_workspace_bytes(const FaPagedPlan* plan)
{
    int device = 0, sms = 0;
    if (fa_sm100_internal::validate_plan(plan) != FA_STATUS_OK ||
        fa_sm100_internal::current_sm100(&device, &sms) != FA_STATUS_OK)
        return 0;
    return workspace_bytes_of(*plan, sms);
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
    for (int i = 0; i < 10; ++i) {
        if (strides[i] < 0) return FA_STATUS_INVALID_ARGUMENT;
        if (strides[i] & 7) return FA_STATUS_MISALIGNED;
    }
    int device = 0, sms = 0;
    status = fa_sm100_internal::current_sm100(&device, &sms);
    if (status != FA_STATUS_OK) return status;
    if ((status = prepare_paged_device(device)) != FA_STATUS_OK) return status;
    if (plan->num_pages == 0) return FA_STATUS_INVALID_ARGUMENT;
    const size_t needed = workspace_bytes_of(*plan, sms);
    if (workspace_bytes < needed) return FA_STATUS_WORKSPACE;
    if (needed > 0 && workspace == nullptr) return FA_STATUS_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return FA_STATUS_MISALIGNED;
    PagedParams params{};
    params.plan = *plan;
    params.q = static_cast<const __nv_bfloat16*>(q);
    params.o = static_cast<__nv_bfloat16*>(o);
    params.q_token = strides[0];
    params.q_head = strides[1];
    params.o_token = strides[2];
    params.o_head = strides[3];
    params.page_shift = __builtin_ctz(static_cast<unsigned>(plan->page_size));
    params.scale_log2 = fa_default_scale(plan->head_dim) * 1.4426950408889634f;
    params.behind_wide = may_be_wide(*plan) ? 1 : 0;
    params.narrow_follows = may_be_narrow(*plan) ? 1 : 0;
    params.inject_stall = t_armed_stall ? 1 : 0;
    t_armed_stall = false;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = may_be_wide(*plan), narrow = may_be_narrow(*plan);
    PagedMaps maps;
    char* work = static_cast<char*>(workspace);
    if (wide) {
        params.wide_partial = reinterpret_cast<float*>(work);
        params.wide_merges = reinterpret_cast<Merge*>(work + wide_parts(sms, plan->head_dim));
        work += wide_workspace(sms, plan->head_dim);
        const int group = plan->heads / plan->kv_heads;
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(plan->head_dim), static_cast<cuuint64_t>(plan->heads),
                                    static_cast<cuuint64_t>(plan->total_tokens)};
        const cuuint64_t bytes[2] = {static_cast<cuuint64_t>(params.q_head) * 2u, static_cast<cuuint64_t>(params.q_token) * 2u};
        const cuuint32_t box[3] = {64u, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(tokens_per_tile(group))};
        if ((status = fa_sm100_internal::encode_map(&maps.q, q, 3, dims, bytes, box)) != FA_STATUS_OK) return status;
        if ((status = cache_map(&maps.wide_k, k_cache, *plan, strides + 4, kWideKeys)) != FA_STATUS_OK) return status;
        if ((status = cache_map(&maps.wide_v, v_cache, *plan, strides + 7, kWideKeys)) != FA_STATUS_OK) return status;
    }
    if (narrow) {
        params.partial = reinterpret_cast<float*>(work);
        params.merges = reinterpret_cast<Merge*>(work + narrow_parts(sms, *plan));
        if (wide && plan->page_size <= kNarrowKeys) {       // the same boxes
            maps.narrow_k = maps.wide_k;
            maps.narrow_v = maps.wide_v;
        } else {
            if ((status = cache_map(&maps.narrow_k, k_cache, *plan, strides + 4, kNarrowKeys)) != FA_STATUS_OK) return status;
            if ((status = cache_map(&maps.narrow_v, v_cache, *plan, strides + 7, kNarrowKeys)) != FA_STATUS_OK) return status;
        }
    }
    const bool one = narrow_rows(*plan) == 16;
    if (plan->head_dim == 64)
        return one ? launch_attention<64, 1>(maps, params, wide, narrow, sms, s)
                   : launch_attention<64, 2>(maps, params, wide, narrow, sms, s);
    return one ? launch_attention<128, 1>(maps, params, wide, narrow, sms, s)
               : launch_attention<128, 2>(maps, params, wide, narrow, sms, s);
}

}  // extern "C"
