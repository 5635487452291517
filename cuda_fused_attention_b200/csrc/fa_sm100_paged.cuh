// What the paged-cache translation units share: the geometry of attention work
// and how a linear range of it maps back to requests.
//
// A request with n new tokens and a group of G query heads per K/V head has n * G query
// rows per K/V head (row = token * G + head in group). Requests of at most narrow_rows(plan) rows
// go to the narrow kernel, whose unit of work is a 64-key tile; all others to the wide kernel,
// which takes 128-key tiles of blocks of 2 * tokens_per_tile(G) tokens, at two units each (one if the
// block has one Q tile). Each narrow item (one K/V head of a request) and each block is preceded by
// kNarrowGap or kWideGap units without work, about what its set-up and epilogue cost. Without the
// narrow gap 32 ragged requests of up to 4096 keys take 55.0 us instead of 52.4, with two 52.8;
// without the wide one a causal prompt of 8192 tokens (32/8 heads) 484 us instead of 437, with two 453, with six 441.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

#include "fa_sm100_paged.h"

namespace fa_sm100 {

constexpr int kNarrowGap = 1;
constexpr int kWideGap = 4;
constexpr int kNarrowKeys = 64;
constexpr int kWideRows = 128;      // query rows of one tile (tensor-memory lanes)
constexpr int kWideKeys = 128;
static_assert(kWideKeys == 128, "floor_sum_128 counts key tiles");

// plan->schedule: narrow_start[num_seqs + 1], then wide_start[num_seqs + 1]: prefix sums of the
// requests' units for one K/V head.
__host__ __device__ inline long long* narrow_starts(long long* schedule) { return schedule; }
__host__ __device__ inline long long* wide_starts(long long* schedule, int num_seqs) { return schedule + num_seqs + 1; }

// Query rows per K/V head that any request of the plan can have, and the most that go to the narrow
// kernel: 32 where no request has more (drafted tokens), else 16, which its faster variant holds. 16
// requests of 5 to 8 new tokens, 20 to 32 rows, behind up to 8192: 62 us against 71 in the wide kernel, at D = 64 40 against 60.
__host__ __device__ inline long long most_rows(const FaPagedPlan& plan)
{
    return static_cast<long long>(plan.max_new < plan.total_tokens ? plan.max_new : plan.total_tokens) *
           (plan.heads / plan.kv_heads);
}
__host__ __device__ inline int narrow_rows(const FaPagedPlan& plan)
{
    const long long most = most_rows(plan);
    return most > 16 && most <= 32 ? 32 : 16;
}

__host__ __device__ inline int tokens_per_tile(int group) { return kWideRows / group; }

// a / b for a >= 0, b > 0: nearly always in 32 bits, where a division costs a fifth. The kernels find their
// first work with these, before anything else can start.
__host__ __device__ inline long long quotient(long long a, long long b)
{
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}
__host__ __device__ inline long long ceil_div(long long a, long long b) { return quotient(a + b - 1, b); }
__host__ __device__ inline long long key_tiles(long long keys) { return (keys + kWideKeys - 1) >> 7; }

// sum over 0 <= i < n of floor((a * i + b) / 128), a > 0, b >= 0. The terms' sum is exact without the
// floors; what the floors drop, (a * i + b) mod 128, repeats with period 128 / gcd(a, 128), and over one
// period takes each value that is b modulo the gcd once. So fewer terms than a period are added up.
__host__ __device__ inline long long floor_sum_128(long long n, int a, long long b)
{
    int log_gcd = 0;
    while (log_gcd < 7 && (a >> log_gcd & 1) == 0) ++log_gcd;
    const int period = 128 >> log_gcd, gcd = 1 << log_gcd;
    const int rest = static_cast<int>(b & 127);
    long long dropped = (n >> (7 - log_gcd)) * (period * (rest & (gcd - 1)) + gcd * (period * (period - 1) / 2));
    const int left = static_cast<int>(n & (period - 1));
    int partial = 0;
    for (int i = 0; i < left; ++i) partial += (a * i + rest) & 127;
    dropped += partial;
    return (n * b + a * (n * (n - 1) / 2) - dropped) >> 7;
}

// Key tiles of token block u (of `span` tokens) of a request with `cached` + `n` tokens.
__host__ __device__ inline long long wide_tiles_of(long long u, int span, long long cached, int n, bool causal)
{
    const long long end = (u + 1) * span < n ? (u + 1) * span : n;
    return key_tiles(cached + (causal ? end : n));
}

// Units of one of its key tiles: a block of one Q tile takes half the time of a block of two.
__host__ __device__ inline int wide_weight(long long u, int span, int n) { return n - u * span <= span / 2 ? 1 : 2; }

// Units (key tiles and gaps) of the request's first `blocks` token blocks, of which `whole` (n / span) are full.
__host__ __device__ inline long long wide_units_through(long long blocks, int whole, int span, long long cached, int n,
                                                        bool causal)
{
    const long long full = whole < blocks ? whole : blocks;
    const long long tiles = causal ? floor_sum_128(full, span, cached + span + kWideKeys - 1) : full * key_tiles(cached + n);
    return blocks * kWideGap + 2 * tiles + (blocks > full ? wide_weight(whole, span, n) * key_tiles(cached + n) : 0);
}

}  // namespace fa_sm100

namespace fa_sm100_internal {

// The device error word of a paged translation unit on the current device: read (synchronous)
// and cleared. Returns a cudaError_t; *word receives the bits.
int take_plan_error(unsigned int* word);
int take_paged_attention_error(unsigned int* word);

int validate_plan(const FaPagedPlan* plan);
bool page_size_supported(int page_size);

// Launches a kernel that may start before the one in front of it in the stream is done, once that one's CTAs
// all run, so that its own start-up hides (attention of one request over 2048 keys 8.9 -> 8.4 us, plan of 16
// requests 4.5 -> 4.2 us). It calls grid_dependency_wait before it touches memory, and
// grid_dependents_launch for the kernel behind it. One does not wait at its start: the narrow attention kernel behind
// the wide one. That one waited before it let any other start, and what the merging kernel between them
// reads and writes is not the narrow kernel's; it waits at its end, so that the call is done when it is.
template <typename... Args>
int launch_early(void (*kernel)(Args...), int grid, int threads, int shared_bytes, cudaStream_t stream, const Args&... args)
{
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(grid));
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.dynamicSmemBytes = static_cast<size_t>(shared_bytes);
    config.stream = stream;
    config.attrs = &attribute;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, args...);
    if (err != cudaSuccess) cudaGetLastError();     // returned here, not left for the caller's next call
    return static_cast<int>(err);
}

// cudaError_t or FA_STATUS_*: the current device, its SM count, and that it is compute capability 10.x.
int current_sm100(int* device, int* sm_count);

}  // namespace fa_sm100_internal
