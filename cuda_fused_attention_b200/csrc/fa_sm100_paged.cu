// Attention of a step's new tokens over a paged K/V cache (sm_100a).

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "fa_sm100_paged.h"
#include "fa_sm100_paged.cuh"

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
};

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
    if (kv < n) return;
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

extern "C" {

size_t fa_sm100_paged_workspace_bytes(const FaPagedPlan* plan)
{
    (void)plan;
    return 0;
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
    (void)workspace;
    if (workspace_bytes < fa_sm100_paged_workspace_bytes(plan)) return FA_STATUS_WORKSPACE;
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
    const long long rows = static_cast<long long>(plan->total_tokens) * plan->heads;
    const long long blocks = (rows + 3) / 4;
    if (blocks > INT_MAX) return FA_STATUS_INVALID_ARGUMENT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (plan->head_dim == 64) paged_rows_kernel<64><<<static_cast<unsigned>(blocks), 128, 0, s>>>(params);
    else paged_rows_kernel<128><<<static_cast<unsigned>(blocks), 128, 0, s>>>(params);
    return static_cast<int>(cudaGetLastError());
}

}  // extern "C"
