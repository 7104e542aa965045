// Log probabilities of given tokens, entropy and the most probable entries of rows of logits.
//
// With m = max x, d = x - m, Z = sum e^d: log p = d - log Z, entropy = log Z - (sum e^d d) / Z.  The maximal entry's own 1 is kept out of the sum, Z = 1 + z
// and log Z = log1p(z): when that entry holds nearly all of the mass, its log probability and the entropy are tiny and keep their digits.
#include "paged.cuh"
#include "tma.cuh"

namespace runit {
namespace lp {

using pg::to_f32;

struct Args {
    const void* x;
    const int32_t* tokens;
    float *logprob, *entropy, *top_logprobs;
    int32_t* top_ids;
    uint32_t ld, n, k;
};

constexpr uint32_t kThreads = 512;

// Order of the logits as integers: NaN before everything, one zero.
__device__ __forceinline__ uint32_t order(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float log_of(float d, float logz) { return d == -INFINITY ? -INFINITY : d - logz; }

// The plainest form: a block per row; a pass for the maximum, one for the sums, one for each of the k entries.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const Args a) {
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ unsigned long long best[kThreads / 32];
    __shared__ float part[2][kThreads / 32];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x;
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.ld;
    // the first entry behind `last` in descending order, equal ones by index
    auto next = [&](unsigned long long last) {
        unsigned long long b = 0;
        for (uint32_t i = tid; i < a.n; i += kThreads) {
            const unsigned long long key = ((unsigned long long)order(to_f32(x[i])) << 32) | (0xFFFFFFFFu - i);
            if (key < last && key > b) b = key;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long t = __shfl_xor_sync(0xffffffffu, b, o);
            b = t > b ? t : b;
        }
        __syncthreads();
        if (lane == 0) best[warp] = b;
        __syncthreads();
        for (uint32_t w = 0; w < kThreads / 32; w++) b = best[w] > b ? best[w] : b;
        return b;
    };
    const unsigned long long top = next(~0ull);
    const float m = to_f32(x[0xFFFFFFFFu - (uint32_t)top]);
    const bool none = m == -INFINITY;
    float z = 0.f, e = 0.f;
    for (uint32_t i = tid; i < a.n; i += kThreads) {
        const float v = to_f32(x[i]), d = none ? 0.f : v - m, p = expf(d);
        if (i != 0xFFFFFFFFu - (uint32_t)top) z += p;
        e += p * (d < -200.f ? -200.f : d);
    }
    for (int o = 16; o > 0; o >>= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, o);
        e += __shfl_xor_sync(0xffffffffu, e, o);
    }
    if (lane == 0) { part[0][warp] = z; part[1][warp] = e; }
    __syncthreads();
    z = e = 0.f;
    for (uint32_t w = 0; w < kThreads / 32; w++) { z += part[0][w]; e += part[1][w]; }
    const float logz = log1pf(z);
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = none ? 0.f : logz - e / (1.f + z);
        if (a.tokens) {
            const int32_t t = a.tokens[row];
            a.logprob[row] = (uint32_t)t >= a.n ? 0.f : none ? -INFINITY : log_of(to_f32(x[t]) - m, logz);
        }
    }
    unsigned long long at = top;
    for (uint32_t i = 0; i < a.k; i++) {
        if (i) at = next(at);
        if (tid == 0) {
            const uint32_t id = 0xFFFFFFFFu - (uint32_t)at;
            a.top_ids[(size_t)row * a.k + i] = (int32_t)id;
            a.top_logprobs[(size_t)row * a.k + i] = none ? -INFINITY : log_of(to_f32(x[id]) - m, logz);
        }
    }
}

}  // namespace lp
}  // namespace runit

using namespace runit;

extern "C" int32_t runit_token_logprobs(runit_ctx_t* ctx, const void* logits, int32_t type, uint32_t ld, uint32_t n, uint32_t rows, const void* tokens,
                                        void* logprob, void* entropy, uint32_t k, void* top_ids, void* top_logprobs) {
    if (!ctx) return RUNIT_ERR_BAD_ARG;
    RUNIT_REQUIRE(ctx, type >= RUNIT_TYPE_F32 && type <= RUNIT_TYPE_BF16, "token_logprobs: type %d", type);
    RUNIT_REQUIRE(ctx, logits && n > 0 && rows > 0 && ld >= n && n <= 0x7FFFFFFFu && rows <= 0x7FFFFFFFu, "token_logprobs: null logits, n=%u, rows=%u or ld=%u", n, rows, ld);
    RUNIT_REQUIRE(ctx, runit_aligned(logits, type == RUNIT_TYPE_F32 ? 4 : 2), "token_logprobs: misaligned logits");
    RUNIT_REQUIRE(ctx, (tokens != nullptr) == (logprob != nullptr), "token_logprobs: tokens and logprob come together");
    RUNIT_REQUIRE(ctx, k <= 32 && k <= n && (k > 0) == (top_ids != nullptr) && (k > 0) == (top_logprobs != nullptr), "token_logprobs: k=%u must be at most 32 and n, with top_ids and top_logprobs", k);
    RUNIT_REQUIRE(ctx, logprob || entropy || k > 0, "token_logprobs: nothing is asked for");
    RUNIT_REQUIRE(ctx, runit_aligned(tokens, 4) && runit_aligned(logprob, 4) && runit_aligned(entropy, 4) && runit_aligned(top_ids, 4) && runit_aligned(top_logprobs, 4),
                  "token_logprobs: misaligned tokens or results");
    const lp::Args a{logits, (const int32_t*)tokens, (float*)logprob, (float*)entropy, (float*)top_logprobs, (int32_t*)top_ids, ld, n, k};
    if (type == RUNIT_TYPE_F32) runit_launch_chain(ctx, lp::token_logprobs_kernel<float>, dim3(rows), dim3(lp::kThreads), a);
    else if (type == RUNIT_TYPE_F16) runit_launch_chain(ctx, lp::token_logprobs_kernel<__half>, dim3(rows), dim3(lp::kThreads), a);
    else runit_launch_chain(ctx, lp::token_logprobs_kernel<__nv_bfloat16>, dim3(rows), dim3(lp::kThreads), a);
    return runit_after_launch(ctx, "token_logprobs");
}
