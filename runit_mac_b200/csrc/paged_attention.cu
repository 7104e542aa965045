// Attention of a batch of sequences over a paged cache: out_i = sum_j softmax_j(s_ij) v_j over the positions j that row i sees, s_ij = scale q_i . k_j,
// then cap * tanh(s / cap), then minus slope * (i - j).
#include "gemv_common.cuh"
#include "paged.cuh"
#include "tma.cuh"

namespace runit {
namespace pg {

struct AttnArgs {
    Cache c;
    const void* q;
    void* out;
    const float* slopes;
    uint32_t ldq, ldo, window;
    float scale, cap;
};

// The plainest form: a block per row and query head, four warps that take its keys in turn, a lane 2 or 4 of the dimensions.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attention_kernel(const AttnArgs a) {
    grid_dependency_wait();
    grid_launch_dependents();
    constexpr int E = HD / 32;
    __shared__ float sm[4], sl[4], so[4][HD];
    const Cache& c = a.c;
    const uint32_t row = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t s = 0;
    for (uint32_t i0 = 1; i0 <= c.n_seqs; i0 += 128) {
        const uint32_t i = i0 + threadIdx.x;
        s += __syncthreads_count(i <= c.n_seqs && c.q_start[i] <= (int32_t)row);
    }
    if (s >= c.n_seqs) return;
    const Seq q = sequence(c, s);
    const uint32_t back = q.row0 + q.n - row;
    if (row < q.row0 || back > q.n) return;
    const uint32_t end = q.len >= back ? q.len - back + 1 : 0, beg = a.window && end > a.window ? end - a.window : 0;
    const T* qp = reinterpret_cast<const T*>(a.q) + (size_t)row * a.ldq + (size_t)head * HD + lane * E;
    float x[E], o[E], m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; e++) { x[e] = to_f32(qp[e]); o[e] = 0.f; }
    const float slope = a.slopes ? a.slopes[head] : 0.f;
    for (uint32_t j = beg + warp; j < end; j += 4) {
        bool ok;
        const size_t at = page_row(c, c.table + (j < c.shared ? 0 : (size_t)s * c.table_ld), j, head / c.group, &ok) + lane * E;
        float t = 0.f;
        for (int e = 0; e < E; e++) t = fmaf(x[e], to_f32(reinterpret_cast<const T*>(c.k)[at + e]), t);
        for (int d = 16; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
        t *= a.scale;
        if (a.cap != 0.f) t = a.cap * tanhf(t / a.cap);
        t -= slope * (float)(end - 1 - j);
        const float top = fmaxf(m, t), old = m == -INFINITY ? 0.f : expf(m - top), p = expf(t - top);
        l = fmaf(l, old, p);
        for (int e = 0; e < E; e++) o[e] = fmaf(o[e], old, p * to_f32(reinterpret_cast<const T*>(c.v)[at + e]));
        m = top;
    }
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
    for (int e = 0; e < E; e++) so[warp][lane * E + e] = o[e];
    __syncthreads();
    if (threadIdx.x < HD) {
        const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
        float num = 0.f, den = 0.f;
        for (int w = 0; w < 4; w++) {
            const float f = sm[w] == -INFINITY ? 0.f : expf(sm[w] - top);
            num = fmaf(f, so[w][threadIdx.x], num);
            den = fmaf(f, sl[w], den);
        }
        reinterpret_cast<T*>(a.out)[(size_t)row * a.ldo + (size_t)head * HD + threadIdx.x] = from_f32<T>(den == 0.f ? 0.f : num / den);
    }
}

}  // namespace pg
}  // namespace runit

using namespace runit;

extern "C" {

size_t runit_paged_attention_scratch_bytes(const runit_paged_cfg* cfg, const runit_paged_batch* batch) { return pg::why_not(cfg, batch) ? 0 : 1024; }

int32_t runit_paged_attention(runit_ctx_t* ctx, const runit_paged_cfg* cfg, const runit_paged_batch* batch, const void* q, uint32_t ldq, void* out,
                              uint32_t ldo, void* scratch, size_t scratch_bytes) {
    if (!ctx) return RUNIT_ERR_BAD_ARG;
    const char* why = pg::why_not(cfg, batch);
    if (!why) why = pg::why_not_memory(cfg, batch);
    RUNIT_REQUIRE(ctx, !why, "paged_attention: %s", why);
    RUNIT_REQUIRE(ctx, q && out && runit_aligned(q, 16) && runit_aligned(out, 16), "paged_attention: q and out must be 16-byte aligned");
    RUNIT_REQUIRE(ctx, ldq % 8 == 0 && ldo % 8 == 0 && ldq >= (uint64_t)cfg->heads * cfg->dim && ldo >= (uint64_t)cfg->heads * cfg->dim,
                  "paged_attention: ldq=%u, ldo=%u must be multiples of 8, rows of heads * dim at least", ldq, ldo);
    RUNIT_REQUIRE(ctx, scratch && runit_aligned(scratch, 256), "paged_attention: scratch must be 256-byte aligned");
    if (scratch_bytes < runit_paged_attention_scratch_bytes(cfg, batch))
        return runit_fail(ctx, RUNIT_ERR_BUFFER_SIZE, "paged_attention: %zu bytes of scratch, %zu needed", scratch_bytes, runit_paged_attention_scratch_bytes(cfg, batch));
    const pg::AttnArgs a{pg::cache_of(ctx, cfg, batch), q, out, (const float*)cfg->slopes, ldq, ldo, cfg->window, cfg->scale, cfg->cap};
    const dim3 grid(batch->rows, cfg->heads);
    if (cfg->type == RUNIT_TYPE_F16) {
        if (cfg->dim == 128) runit_launch_chain(ctx, pg::paged_attention_kernel<__half, 128>, grid, dim3(128), a);
        else runit_launch_chain(ctx, pg::paged_attention_kernel<__half, 64>, grid, dim3(128), a);
    } else {
        if (cfg->dim == 128) runit_launch_chain(ctx, pg::paged_attention_kernel<__nv_bfloat16, 128>, grid, dim3(128), a);
        else runit_launch_chain(ctx, pg::paged_attention_kernel<__nv_bfloat16, 64>, grid, dim3(128), a);
    }
    return runit_after_launch(ctx, "paged_attention");
}

}  // extern "C"
