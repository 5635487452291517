// Paged-cache plan and rotary kernels (sm_100a): block tables and slot maps built
// from request lengths, rotary positions, and the write of K and V to cache slots.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "fa_sm100_paged.h"
#include "fa_sm100_paged.cuh"
#include "fa_sm100_ptx.cuh"

namespace fa_sm100 {

__device__ unsigned int g_plan_error_word;

__device__ __forceinline__ void record_plan_error(unsigned int bits) { atomicOr(&g_plan_error_word, bits); }

// =============================================================================
// Plan
// =============================================================================
// Three prefix sums over the requests (new tokens, new pages, attention units), then one slot
// per new token and one table entry per new page. The bytes are few (16 per request, 8 per token,
// 8 per new page), so the time is launch and latency: everything is one launch. Every CTA runs
// the scan over all requests, 512 at a time, and after each 512 serves its share of their tokens
// and pages, found by binary search in shared memory; the CTAs never wait for one another. A new
// page's id is taken from the free list, not from the table that another CTA may be writing. Measured
// (B200): 4.4 us for 16 decoding requests, 8.0 us for 512 requests with 99k new tokens.
constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanTokensPerCta = 2048;     // tokens before another CTA is launched (99k tokens: 7.9 us; 4096: 10.0, 1024: 7.5, 512: 6.4)

struct PlanParams {
    FaPagedPlan plan;
    const int* cached;
    const int* fresh;               // new_lens
    const int* free_pages;
    int num_free;
    const int* free_start;
};

struct PlanSums {
    long long tokens, pages, narrow, wide;
};

__device__ __forceinline__ long long warp_inclusive(long long v, int lane)
{
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long other = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += other;
    }
    return v;
}

__global__ void __launch_bounds__(kPlanThreads)
plan_kernel(const __grid_constant__ PlanParams p)
{
    grid_dependents_launch();
    grid_dependency_wait();
    const FaPagedPlan& plan = p.plan;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int ps = plan.page_size;
    const int shift = __ffs(ps) - 1;
    const int group = plan.heads / plan.kv_heads;
    const int span = 2 * tokens_per_tile(group);
    const bool first_cta = blockIdx.x == 0;

    __shared__ PlanSums warp_sums[kPlanWarps];
    __shared__ int s_start[kPlanThreads + 1];       // packed row of each request of this round
    __shared__ int s_page[kPlanThreads];            // new pages before each request of this round
    __shared__ unsigned long long s_unplaced;       // pages of this round's requests that have no rows
    __shared__ int s_cached[kPlanThreads];          // cached tokens, -1 for a request with invalid lengths
    long long* narrow = narrow_starts(plan.schedule);
    long long* wide = wide_starts(plan.schedule, plan.num_seqs);

    const long long free_start = p.free_start ? *p.free_start : 0;
    PlanSums carry = {0, 0, 0, 0};
    for (int base = 0; base < plan.num_seqs; base += kPlanThreads) {
        const int b = base + tid;
        long long cached = 0, n = 0, need = 0, narrow_units = 0, wide_units = 0;
        bool valid = false;
        if (b < plan.num_seqs) {
            cached = p.cached[b];
            n = p.fresh[b];
            valid = cached >= 0 && n >= 0 && n <= plan.total_tokens && n <= plan.max_new &&
                    cached + n <= static_cast<long long>(plan.table_width) * ps;
            if (!valid && first_cta) record_plan_error(FA_ERROR_BAD_LENGTH);
            // A request with invalid lengths keeps its place on the token axis if that is known.
            if (n < 0) n = 0;
            if (n > plan.total_tokens) n = plan.total_tokens;
        }
        if (valid) {
            const long long kv = cached + n;
            need = ((kv + ps - 1) >> shift) - ((cached + ps - 1) >> shift);
        }
        PlanSums sum;
        sum.tokens = warp_inclusive(n, lane);
        sum.pages = warp_inclusive(need, lane);
        // The tokens of requests past total_tokens have no rows: such a request gets no work.
        if (lane == 31) warp_sums[warp] = {sum.tokens, sum.pages, 0, 0};
        if (tid == 0) s_unplaced = 0;
        __syncthreads();
        long long tokens_before = carry.tokens + sum.tokens - n, pages_before = carry.pages + sum.pages - need;
        long long round_tokens = 0, round_pages = 0;
        for (int w = 0; w < kPlanWarps; ++w) {
            if (w < warp) {
                tokens_before += warp_sums[w].tokens;
                pages_before += warp_sums[w].pages;
            }
            round_tokens += warp_sums[w].tokens;
            round_pages += warp_sums[w].pages;
        }
        const long long total = plan.total_tokens;
        const bool fits = tokens_before + n <= total;
        if (!fits && first_cta && b < plan.num_seqs) record_plan_error(FA_ERROR_BAD_LENGTH);
        // Nor does it get pages. Requests behind it have no rows either, so the sums before those that fit stand.
        if (!fits && need > 0) atomicAdd(&s_unplaced, static_cast<unsigned long long>(need));
        if (valid && fits && n > 0) {
            if (n * group <= narrow_rows(plan)) narrow_units = kNarrowGap + ceil_div(cached + n, kNarrowKeys);
            else
                wide_units = wide_units_through(ceil_div(n, span), static_cast<int>(n) / span, span, cached, static_cast<int>(n),
                                                plan.causal != 0);
        }
        s_start[tid] = static_cast<int>(tokens_before < total ? tokens_before : total);
        s_page[tid] = static_cast<int>(pages_before - carry.pages < INT_MAX ? pages_before - carry.pages : INT_MAX);
        s_cached[tid] = valid && fits ? static_cast<int>(cached) : -1;
        if (tid == 0) {
            const long long end = carry.tokens + round_tokens;
            s_start[kPlanThreads] = static_cast<int>(end < total ? end : total);
        }
        if (first_cta) {
            // Only one CTA writes the per-request arrays, so only it needs the units' sums.
            sum.narrow = warp_inclusive(narrow_units, lane);
            sum.wide = warp_inclusive(wide_units, lane);
            __syncthreads();
            if (lane == 31) { warp_sums[warp].narrow = sum.narrow; warp_sums[warp].wide = sum.wide; }
            __syncthreads();
            long long narrow_before = carry.narrow + sum.narrow - narrow_units;
            long long wide_before = carry.wide + sum.wide - wide_units;
            for (int w = 0; w < kPlanWarps; ++w) {
                if (w < warp) {
                    narrow_before += warp_sums[w].narrow;
                    wide_before += warp_sums[w].wide;
                }
                carry.narrow += warp_sums[w].narrow;
                carry.wide += warp_sums[w].wide;
            }
            if (b < plan.num_seqs) {
                plan.query_start[b] = s_start[tid];
                plan.kv_lens[b] = valid && fits ? static_cast<int>(cached + n) : 0;
                narrow[b] = narrow_before;
                wide[b] = wide_before;
            }
        }
        __syncthreads();

        // This round's tokens: t in [s_start[0], s_start[last]), a contiguous share per CTA.
        const int first = s_start[0], count = s_start[kPlanThreads] - first;
        const int share = (count + gridDim.x - 1) / static_cast<int>(gridDim.x);
        const int lo = first + static_cast<int>(min(static_cast<long long>(share) * blockIdx.x, static_cast<long long>(count)));
        const int hi = min(first + count, lo + share);
        for (int t = lo + tid; t < hi; t += kPlanThreads) {
            int r = 0;
#pragma unroll
            for (int step = kPlanThreads / 2; step > 0; step >>= 1)
                if (s_start[r + step] <= t) r += step;
            const int cached_r = s_cached[r];
            const long long pos = static_cast<long long>(cached_r) + (t - s_start[r]);
            int slot = -1;
            if (cached_r >= 0 && pos < static_cast<long long>(plan.table_width) * ps) {
                const int index = static_cast<int>(pos >> shift);
                const int have = static_cast<int>((static_cast<long long>(cached_r) + ps - 1) >> shift);
                int page = -1;
                if (index < have) {
                    page = plan.block_table[static_cast<long long>(base + r) * plan.table_stride + index];
                    if (page < 0 || page >= plan.num_pages) {
                        record_plan_error(FA_ERROR_BAD_PAGE);
                        page = -1;
                    }
                } else {
                    // A free page that is missing or outside the cache is recorded where it is handed out.
                    const long long from = free_start + carry.pages + s_page[r] + (index - have);
                    if (from >= 0 && from < p.num_free) page = p.free_pages[from];
                    if (page < 0 || page >= plan.num_pages) page = -1;
                }
                if (page >= 0) slot = page * ps + static_cast<int>(pos & (ps - 1));
            }
            plan.positions[t] = cached_r >= 0 ? static_cast<int>(pos) : 0;
            plan.slots[t] = slot;
        }

        // This round's new pages: at most one per 16 rows and one per request, so k stays far below 2^31.
        round_pages -= static_cast<long long>(s_unplaced);
        const int pages = static_cast<int>(round_pages);
        for (int k = blockIdx.x * kPlanThreads + tid; k < pages; k += gridDim.x * kPlanThreads) {
            int r = 0;
#pragma unroll
            for (int step = kPlanThreads / 2; step > 0; step >>= 1)
                if (s_page[r + step] <= k) r += step;
            if (s_cached[r] < 0) continue;
            const int have = static_cast<int>((static_cast<long long>(s_cached[r]) + ps - 1) >> shift);
            const long long from = free_start + carry.pages + k;
            // Where no page is to be had the entry says so: what it held before may be another request's page.
            int page = -1;
            if (from < 0 || from >= p.num_free) {
                record_plan_error(FA_ERROR_OUT_OF_PAGES);
            } else {
                page = p.free_pages[from];
                if (page < 0 || page >= plan.num_pages) {
                    record_plan_error(FA_ERROR_BAD_PAGE);
                    page = -1;
                }
            }
            plan.block_table[static_cast<long long>(base + r) * plan.table_stride + have + (k - s_page[r])] = page;
        }
        carry.tokens += round_tokens;
        carry.pages += round_pages;
        __syncthreads();
    }

    if (first_cta && tid == 0) {
        plan.query_start[plan.num_seqs] =
            static_cast<int>(carry.tokens < plan.total_tokens ? carry.tokens : plan.total_tokens);
        narrow[plan.num_seqs] = carry.narrow;
        wide[plan.num_seqs] = carry.wide;
        *plan.free_cursor = static_cast<int>(free_start + carry.pages);
    }
    // Padding rows behind the last request.
    const long long used = carry.tokens < plan.total_tokens ? carry.tokens : plan.total_tokens;
    for (long long t = used + blockIdx.x * kPlanThreads + tid; t < plan.total_tokens; t += gridDim.x * kPlanThreads) {
        plan.positions[t] = 0;
        plan.slots[t] = -1;
    }
}

// =============================================================================
// Rotary positions, and the append of K and V
// =============================================================================
// Every element is read once and written once, in units of eight pairs (two 16-byte accesses); memory
// bounds it once there is enough of it. An angle is a position times a frequency; far positions need
// more than 24 bits of it, so the product is taken in turns (1 / 2 pi) in 64 bits, its whole turns
// dropped there, and only the rest goes to sincospif. That costs more than a unit's rotation, so
// angles are shared by the heads, in one of two ways:
//   rotary_kernel      a CTA serves a few neighbouring tokens; their angles go through shared memory
//   rotary_long_kernel a thread keeps the angles of one token's unit in registers and walks over
//                      heads; neighbouring threads take neighbouring tokens, so that each head of a
//                      [heads, tokens] tensor is read in long runs
// Measured (B200): append of 6.8k tokens (32/8 heads, D = 128) 31 us, 5.4 TB/s; 32 heads of 16384 tokens
// 45 us, 5.9 TB/s (54 us with rotary_kernel); 2 x 8 heads of 2048 tokens, D = 64, 4.3 us (6.1 with
// rotary_long_kernel); they meet at 8192 tokens of 32 heads, 26.4 us each.
constexpr int kRotaryThreads = 256;
constexpr int kMaxAxes = 4;
constexpr int kMaxTokensPerCta = 4;     // tokens that share a CTA of rotary_kernel

struct RotaryParams {
    const __nv_bfloat16* src[3];        // q, k, v (x alone: q)
    __nv_bfloat16* dst[3];
    long long src_token[3], src_head[3], src_batch;
    long long dst_token[3], dst_head[3], dst_batch;     // k, v of an append: dst_token is the row stride
    long long dst_page[3];
    int rows[3];                        // heads of each
    int batch, tokens;
    int unit_shift;                     // log2 of the 16-element units per row
    int group_shift;                    // rotary_kernel: log2 of the tokens per CTA
    int head_split;                     // rotary_long_kernel: threads that share a token's heads
    int rotary_dim;
    const int* positions;
    long long position_axis, position_batch;
    const float* inv_freq;
    int section_end[kMaxAxes];
    const int* slots;
    int page_shift;
    long long num_slots;
    float sign;                         // -1: inverse rotation
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8])
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 pair = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&pair);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// (cos, sin) of a token's pair.
__device__ __forceinline__ float2 rotary_angle(const RotaryParams& p, int batch, int token, int pair)
{
    int axis = 0;
#pragma unroll
    for (int a = 0; a < kMaxAxes - 1; ++a) axis += pair >= p.section_end[a] ? 1 : 0;
    const int position = p.positions[axis * p.position_axis + batch * p.position_batch + token];
    const double around = static_cast<double>(position) * static_cast<double>(p.inv_freq[pair]) * 0.15915494309189533577;
    float sine, cosine;
    sincospif(2.0f * static_cast<float>(around - rint(around)), &sine, &cosine);
    return make_float2(cosine, p.sign * sine);
}

// A unit's eight pairs turned: x0 and x1 are its two pieces, turn(i) the (cos, sin) of its pairs 2i and 2i + 1.
template <bool kInterleaved, typename Turn>
__device__ __forceinline__ void rotate_unit(uint4& x0, uint4& x1, Turn&& turn)
{
    float a[8], b[8], u[8], w[8];
    unpack8(x0, a);
    unpack8(x1, b);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float4 two = turn(i / 2);
        if (kInterleaved) {
            float(&v)[8] = i < 4 ? a : b;
            float(&out)[8] = i < 4 ? u : w;
            const int q = 2 * (i & 3);
            out[q] = v[q] * two.x - v[q + 1] * two.y;
            out[q + 1] = v[q + 1] * two.x + v[q] * two.y;
            out[q + 2] = v[q + 2] * two.z - v[q + 3] * two.w;
            out[q + 3] = v[q + 3] * two.z + v[q + 2] * two.w;
        } else {
            u[i] = a[i] * two.x - b[i] * two.y;
            w[i] = b[i] * two.x + a[i] * two.y;
            u[i + 1] = a[i + 1] * two.z - b[i + 1] * two.w;
            w[i + 1] = b[i + 1] * two.z + a[i + 1] * two.w;
        }
    }
    x0 = pack8(u);
    x1 = pack8(w);
}

template <bool kAppend, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads, 6)
rotary_kernel(const __grid_constant__ RotaryParams p)
{
    grid_dependents_launch();
    grid_dependency_wait();
    __shared__ __align__(16) float2 turn[kMaxTokensPerCta][64];
    __shared__ long long slots[kMaxTokensPerCta];
    const int group = 1 << p.group_shift;
    const int blocks_per_batch = (p.tokens + group - 1) >> p.group_shift;
    const int batch = kAppend ? 0 : static_cast<int>(blockIdx.x) / blocks_per_batch;
    const int token0 = (static_cast<int>(blockIdx.x) - batch * blocks_per_batch) << p.group_shift;
    const int tokens = min(group, p.tokens - token0);
    const int pairs = p.rotary_dim / 2;

    // An item is a unit of a row. Neighbouring threads take the units of a row, then the rows that are
    // neighbours in memory: the next head of a packed token, the next token of a [heads, tokens] tensor.
    const int rows = p.rows[0] + (kAppend ? p.rows[1] + p.rows[2] : 0);
    const int total = (kAppend ? tokens : group) * rows << p.unit_shift;
    const int unit = threadIdx.x & ((1 << p.unit_shift) - 1);       // the same for all of a thread's items
    const bool turns = unit < p.rotary_dim / 16;
    // The unit's two 8-element pieces: the two halves of its pairs, or 16 neighbours.
    const int lo = turns && !kInterleaved ? 8 * unit : 16 * unit;
    const int hi = turns && !kInterleaved ? pairs + 8 * unit : 16 * unit + 8;
    int tok, head, which;           // of the item at hand
    auto locate = [&](int index) -> bool {
        const int item = index >> p.unit_shift;
        which = 0;
        if (kAppend) {
            tok = item / rows;
            head = item - tok * rows;
            if (head >= p.rows[0]) { head -= p.rows[0]; which = 1; }
            if (which == 1 && head >= p.rows[1]) { head -= p.rows[1]; which = 2; }
            return index < total;
        }
        tok = item & (group - 1);
        head = item >> p.group_shift;
        return index < total && tok < tokens;
    };
    uint4 x0, x1;
    auto load = [&]() {
        const __nv_bfloat16* src = p.src[which] + batch * p.src_batch + (token0 + tok) * p.src_token[which] +
                                   head * p.src_head[which];
        x0 = *reinterpret_cast<const uint4*>(src + (which == 2 ? 16 * unit : lo));
        x1 = *reinterpret_cast<const uint4*>(src + (which == 2 ? 16 * unit + 8 : hi));
    };

    // The first rows are on their way while the angles are computed.
    if (locate(threadIdx.x)) load();
    if (kAppend && threadIdx.x < tokens) {
        long long slot = p.slots[token0 + threadIdx.x];
        if (slot >= p.num_slots) {
            record_plan_error(FA_ERROR_BAD_PAGE);
            slot = -1;
        }
        slots[threadIdx.x] = slot;
    }
    for (int i = threadIdx.x; i < tokens * pairs; i += kRotaryThreads)
        turn[i / pairs][i % pairs] = rotary_angle(p, batch, token0 + i / pairs, i % pairs);
    __syncthreads();

    for (int index = threadIdx.x; index < total; index += kRotaryThreads) {
        if (!locate(index)) continue;
        const long long slot = kAppend ? slots[tok] : 0;
        if (slot < 0) continue;
        if (index != threadIdx.x) load();
        const bool copied = kAppend && which == 2;
        if (turns && !copied) {
            const float4* cs = reinterpret_cast<const float4*>(&turn[tok][8 * unit]);
            rotate_unit<kInterleaved>(x0, x1, [&](int i) { return cs[i]; });
        }
        __nv_bfloat16* dst = p.dst[which] + head * p.dst_head[which];
        if (kAppend && which > 0)
            dst += (slot >> p.page_shift) * p.dst_page[which] + (slot & ((1LL << p.page_shift) - 1)) * p.dst_token[which];
        else
            dst += batch * p.dst_batch + (token0 + tok) * p.dst_token[which];
        *reinterpret_cast<uint4*>(dst + (copied ? 16 * unit : lo)) = x0;
        *reinterpret_cast<uint4*>(dst + (copied ? 16 * unit + 8 : hi)) = x1;
    }
}

template <bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads)
rotary_long_kernel(const __grid_constant__ RotaryParams p)
{
    grid_dependents_launch();
    grid_dependency_wait();
    const long long index = static_cast<long long>(blockIdx.x) * kRotaryThreads + threadIdx.x;
    const int unit = static_cast<int>(index) & ((1 << p.unit_shift) - 1);
    const long long all = static_cast<long long>(p.tokens) * p.batch, rest = index >> p.unit_shift;
    const int part = static_cast<int>(rest / all);
    if (part >= p.head_split) return;
    const long long flat = rest - part * all;
    const int batch = static_cast<int>(flat / p.tokens), token = static_cast<int>(flat - static_cast<long long>(batch) * p.tokens);
    const int pairs = p.rotary_dim / 2;
    const bool turns = unit < p.rotary_dim / 16;
    const int lo = turns && !kInterleaved ? 8 * unit : 16 * unit;
    const int hi = turns && !kInterleaved ? pairs + 8 * unit : 16 * unit + 8;
    float4 cs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!turns) break;
        const float2 even = rotary_angle(p, batch, token, 8 * unit + 2 * i), odd = rotary_angle(p, batch, token, 8 * unit + 2 * i + 1);
        cs[i] = make_float4(even.x, even.y, odd.x, odd.y);
    }
    const __nv_bfloat16* src = p.src[0] + batch * p.src_batch + token * p.src_token[0];
    __nv_bfloat16* dst = p.dst[0] + batch * p.dst_batch + token * p.dst_token[0];
    for (int head = part; head < p.rows[0]; head += p.head_split) {
        uint4 x0 = *reinterpret_cast<const uint4*>(src + head * p.src_head[0] + lo);
        uint4 x1 = *reinterpret_cast<const uint4*>(src + head * p.src_head[0] + hi);
        if (turns) rotate_unit<kInterleaved>(x0, x1, [&](int i) { return cs[i]; });
        *reinterpret_cast<uint4*>(dst + head * p.dst_head[0] + lo) = x0;
        *reinterpret_cast<uint4*>(dst + head * p.dst_head[0] + hi) = x1;
    }
}

}  // namespace fa_sm100

// =============================================================================
// Host side
// =============================================================================
namespace {

using namespace fa_sm100;

// FA_STATUS_OK if all strides are multiples of 8 and none is negative.
int check_strides(const long long* strides, int count)
{
    for (int i = 0; i < count; ++i) {
        if (strides[i] < 0) return FA_STATUS_INVALID_ARGUMENT;
        if (strides[i] & 7) return FA_STATUS_MISALIGNED;
    }
    return FA_STATUS_OK;
}

bool misaligned(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) != 0; }

int fill_sections(RotaryParams& params, const int* sections, int axes, int rotary_dim)
{
    int end = 0;
    for (int a = 0; a < kMaxAxes; ++a) {
        if (a < axes) {
            if (sections[a] < 0 || sections[a] > rotary_dim / 2) return FA_STATUS_INVALID_ARGUMENT;
            end += sections[a];
        }
        params.section_end[a] = end;
    }
    return end == rotary_dim / 2 ? FA_STATUS_OK : FA_STATUS_INVALID_ARGUMENT;
}

// Units of one head per SM from which rotary_embed takes the long kernel.
constexpr long long kLongUnits = 512;

template <bool kAppend>
int launch_rotary(RotaryParams& params, bool interleaved, cudaStream_t stream)
{
    int device = 0, sms = 0;
    const int status = fa_sm100_internal::current_sm100(&device, &sms);
    if (status != FA_STATUS_OK) return status;
    const long long tokens = static_cast<long long>(params.tokens) * params.batch;
    const int rows = params.rows[0] + (kAppend ? params.rows[1] + params.rows[2] : 0);
    if (tokens == 0 || rows == 0) return FA_STATUS_OK;
    if (tokens > INT_MAX || (static_cast<long long>(rows) << 7) > INT_MAX) return FA_STATUS_INVALID_ARGUMENT;
    const long long units = tokens << params.unit_shift;        // of one head
    if (!kAppend && units >= kLongUnits * static_cast<long long>(sms)) {
        // Heads are shared out until the threads fill the GPU once (2048 per SM).
        const long long split = (2048LL * sms + units - 1) / units;
        params.head_split = static_cast<int>(split < rows ? split : rows);
        const long long blocks = ceil_div(units * params.head_split, kRotaryThreads);
        if (blocks > INT_MAX) return FA_STATUS_INVALID_ARGUMENT;
        return fa_sm100_internal::launch_early(interleaved ? rotary_long_kernel<true> : rotary_long_kernel<false>,
                                               static_cast<int>(blocks), kRotaryThreads, 0, stream, params);
    }
    // Tokens share a CTA (and its set-up) once the CTAs would fill the GPU without it, four per SM.
    params.group_shift = 0;
    while ((2 << params.group_shift) <= kMaxTokensPerCta && (tokens >> (params.group_shift + 1)) >= 4LL * sms)
        ++params.group_shift;
    const long long blocks = ceil_div(params.tokens, 1LL << params.group_shift) * params.batch;
    if (blocks > INT_MAX) return FA_STATUS_INVALID_ARGUMENT;
    return fa_sm100_internal::launch_early(interleaved ? rotary_kernel<kAppend, true> : rotary_kernel<kAppend, false>,
                                           static_cast<int>(blocks), kRotaryThreads, 0, stream, params);
}

}  // namespace

namespace fa_sm100_internal {

int take_plan_error(unsigned int* word)
{
    cudaError_t err = cudaMemcpyFromSymbol(word, g_plan_error_word, sizeof(*word));
    const unsigned int zero = 0;
    if (err == cudaSuccess && *word != 0) err = cudaMemcpyToSymbol(g_plan_error_word, &zero, sizeof(zero));
    return static_cast<int>(err);
}

}  // namespace fa_sm100_internal

extern "C" {

size_t fa_sm100_paged_schedule_bytes(int num_seqs)
{
    return num_seqs < 0 ? 0 : 2 * (static_cast<size_t>(num_seqs) + 1) * sizeof(long long);
}

int fa_sm100_paged_plan(const FaPagedPlan* plan, const int* cached_lens, const int* new_lens, const int* free_pages,
                        int num_free, const int* free_start, void* stream)
{
    int status = fa_sm100_internal::validate_plan(plan);
    if (status != FA_STATUS_OK) return status;
    if (num_free < 0 || (num_free > 0 && free_pages == nullptr)) return FA_STATUS_INVALID_ARGUMENT;
    if (plan->num_seqs > 0 && (cached_lens == nullptr || new_lens == nullptr)) return FA_STATUS_INVALID_ARGUMENT;
    int device = 0, sms = 0;
    status = fa_sm100_internal::current_sm100(&device, &sms);
    if (status != FA_STATUS_OK) return status;
    PlanParams params{*plan, cached_lens, new_lens, free_pages, num_free, free_start};
    long long blocks = ceil_div(plan->total_tokens, kPlanTokensPerCta);
    if (blocks < 1) blocks = 1;
    if (blocks > sms) blocks = sms;
    return fa_sm100_internal::launch_early(plan_kernel, static_cast<int>(blocks), kPlanThreads, 0,
                                           static_cast<cudaStream_t>(stream), params);
}

int fa_sm100_rotary(const void* x, const long long* x_strides, void* out, const long long* out_strides, int batch,
                    int heads, int seq_len, int head_dim, const int* positions, const long long* position_strides,
                    const float* inv_freq, int rotary_dim, const int* sections, int axes, int interleaved, int inverse,
                    void* stream)
{
    if (batch < 0 || heads < 0 || seq_len < 0 || x_strides == nullptr || out_strides == nullptr ||
        position_strides == nullptr || sections == nullptr || axes < 1 || axes > kMaxAxes)
        return FA_STATUS_INVALID_ARGUMENT;
    if (head_dim != 64 && head_dim != 128) return FA_STATUS_UNSUPPORTED;
    if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 16) return FA_STATUS_INVALID_ARGUMENT;
    RotaryParams params{};
    int status = fill_sections(params, sections, axes, rotary_dim);
    if (status != FA_STATUS_OK) return status;
    if (batch == 0 || heads == 0 || seq_len == 0) return FA_STATUS_OK;
    if (x == nullptr || out == nullptr || positions == nullptr || inv_freq == nullptr) return FA_STATUS_INVALID_ARGUMENT;
    if (misaligned(x) || misaligned(out)) return FA_STATUS_MISALIGNED;
    if ((status = check_strides(x_strides, 3)) != FA_STATUS_OK || (status = check_strides(out_strides, 3)) != FA_STATUS_OK)
        return status;
    params.src[0] = static_cast<const __nv_bfloat16*>(x);
    params.dst[0] = static_cast<__nv_bfloat16*>(out);
    params.src_batch = x_strides[0];
    params.src_head[0] = x_strides[1];
    params.src_token[0] = x_strides[2];
    params.dst_batch = out_strides[0];
    params.dst_head[0] = out_strides[1];
    params.dst_token[0] = out_strides[2];
    params.rows[0] = heads;
    params.batch = batch;
    params.tokens = seq_len;
    params.unit_shift = head_dim == 64 ? 2 : 3;
    params.rotary_dim = rotary_dim;
    params.positions = positions;
    params.position_axis = position_strides[0];
    params.position_batch = position_strides[1];
    params.inv_freq = inv_freq;
    params.sign = inverse ? -1.0f : 1.0f;
    return launch_rotary<false>(params, interleaved != 0, static_cast<cudaStream_t>(stream));
}

int fa_sm100_rotary_append(const void* q, const void* k, const void* v, void* q_out, void* k_cache, void* v_cache,
                           const long long* strides, int tokens, int heads, int kv_heads, int head_dim, int page_size,
                           int num_pages, const int* positions, long long position_stride, const int* slots,
                           const float* inv_freq, int rotary_dim, const int* sections, int axes, int interleaved,
                           void* stream)
{
    if (tokens < 0 || heads < 1 || kv_heads < 1 || strides == nullptr || sections == nullptr || axes < 1 ||
        axes > kMaxAxes || num_pages < 0)
        return FA_STATUS_INVALID_ARGUMENT;
    if (head_dim != 64 && head_dim != 128) return FA_STATUS_UNSUPPORTED;
    if (!fa_sm100_internal::page_size_supported(page_size)) return FA_STATUS_UNSUPPORTED;
    if (static_cast<long long>(num_pages) * page_size > INT_MAX) return FA_STATUS_INVALID_ARGUMENT;
    if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 16) return FA_STATUS_INVALID_ARGUMENT;
    RotaryParams params{};
    int status = fill_sections(params, sections, axes, rotary_dim);
    if (status != FA_STATUS_OK) return status;
    if (tokens == 0) return FA_STATUS_OK;
    if (q == nullptr || k == nullptr || v == nullptr || q_out == nullptr || k_cache == nullptr || v_cache == nullptr ||
        positions == nullptr || slots == nullptr || inv_freq == nullptr)
        return FA_STATUS_INVALID_ARGUMENT;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(q_out) || misaligned(k_cache) ||
        misaligned(v_cache))
        return FA_STATUS_MISALIGNED;
    if ((status = check_strides(strides, 14)) != FA_STATUS_OK) return status;
    if (k_cache == v_cache) return FA_STATUS_INVALID_ARGUMENT;
    params.src[0] = static_cast<const __nv_bfloat16*>(q);
    params.src[1] = static_cast<const __nv_bfloat16*>(k);
    params.src[2] = static_cast<const __nv_bfloat16*>(v);
    params.dst[0] = static_cast<__nv_bfloat16*>(q_out);
    params.dst[1] = static_cast<__nv_bfloat16*>(k_cache);
    params.dst[2] = static_cast<__nv_bfloat16*>(v_cache);
    params.src_token[0] = strides[0];
    params.src_head[0] = strides[1];
    params.dst_token[0] = strides[2];
    params.dst_head[0] = strides[3];
    params.src_token[1] = strides[4];
    params.src_head[1] = strides[5];
    params.src_token[2] = strides[6];
    params.src_head[2] = strides[7];
    params.dst_page[1] = strides[8];
    params.dst_head[1] = strides[9];
    params.dst_token[1] = strides[10];
    params.dst_page[2] = strides[11];
    params.dst_head[2] = strides[12];
    params.dst_token[2] = strides[13];
    params.rows[0] = heads;
    params.rows[1] = kv_heads;
    params.rows[2] = kv_heads;
    params.batch = 1;
    params.tokens = tokens;
    params.unit_shift = head_dim == 64 ? 2 : 3;
    params.rotary_dim = rotary_dim;
    params.positions = positions;
    params.position_axis = position_stride;
    params.inv_freq = inv_freq;
    params.slots = slots;
    params.page_shift = __builtin_ctz(static_cast<unsigned>(page_size));
    params.num_slots = static_cast<long long>(num_pages) * page_size;
    params.sign = 1.0f;
    return launch_rotary<true>(params, interleaved != 0, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
