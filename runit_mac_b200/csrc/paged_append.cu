// Rows of a projection on their way into a paged cache: rotation by position, keys and values into the pages, queries out.
//
// y_i = x_i cos a_i - x_{i+h} sin a_i, y_{i+h} = x_i sin a_i + x_{i+h} cos a_i for i < h = rot_dims / 2, a_i = position * freq_i.  The position is an
// integer and freq_i the sum of two floats, so that the angle of a far position keeps its 24 bits (a product of two floats loses as many as the
// position has); from 2^17 on it is formed in 64 bits.  One rounding, at the end.
// Bound: HBM (every value is read once and written once: 7167 rows of 16 + 32 heads of 128 from f32, 264 MB, in 45 to 46 us; a block per row of 192 threads that ask for
// their 128 bytes each before anything else; 128 threads with 4 such pieces 3 more); latency for a few rows.
#include "linear_state.cuh"
#include "paged.cuh"
#include "tma.cuh"

namespace runit {
namespace pg {

constexpr uint32_t kAppendThreads = 192, kAppendItems = 2, kMaxRot = 128;

struct AppendArgs {
    Cache c;
    const void* proj;
    void* q_out;
    const float* freq;
    uint32_t ld, ldq, rot;
};

// eight neighbouring values
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p + 4));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = to_f32(e[i]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = u;
}

// Sine and cosine of the angle of a position from 2^17 on: the turn by what the f32 product was rounded by, which the near ones take, is of the second order, and
// short by 4e-7 at 2^18 and 2e-3 at 2^22; from 2^24 on the position itself is no f32.
__device__ __noinline__ float2 sincos_far(uint32_t pos, float hi, float lo) {
    double s, c;
    sincos((double)pos * ((double)hi + (double)lo), &s, &c);
    return make_float2((float)s, (float)c);
}

// The sequence of a row (as many as have ended at or before it), by all threads of the block; c.n_seqs: nobody's row.
__device__ __forceinline__ uint32_t sequence_of(const Cache& c, uint32_t row) {
    uint32_t s = 0;
    for (uint32_t i0 = 1; i0 <= c.n_seqs; i0 += blockDim.x) {
        const uint32_t i = i0 + threadIdx.x;
        s += __syncthreads_count(i <= c.n_seqs && c.q_start[i] <= (int32_t)row);
    }
    return s;
}

// One block per row.  VEC: items of 16 values, two runs of 8 that the rotation pairs (or 16 neighbours); else pairs of values one by one (rot_dims no
// multiple of 16, or rows that are not 16-byte aligned).
template <typename TP, typename TC, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs a) {
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float cs[kMaxRot / 2], sn[kMaxRot / 2];
    const Cache& c = a.c;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, half = a.rot / 2, dim = c.dim;
    const uint32_t first = a.q_out ? 0 : c.heads, turned = c.heads + c.kv_heads, all = turned + c.kv_heads;
    const TP* x = reinterpret_cast<const TP*>(a.proj) + (size_t)row * a.ld;
    // items of 16 values, kAppendItems a thread at a time; the first ones are asked for ahead of the way to their pages
    const uint32_t per = dim / 16, n = (all - first) * per, pairs = a.rot / 16;
    struct Item {
        uint32_t head, lo;
        bool turn;
    };
    auto item_of = [&](uint32_t i) {
        const uint32_t head = first + i / per, d = i % per;
        const bool turn = head < turned && d < pairs;
        return Item{head, turn ? 8 * d : head < turned ? a.rot + 16 * (d - pairs) : 16 * d, turn};
    };
    float u[kAppendItems][8], v[kAppendItems][8];
    auto ask = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t e = 0; e < kAppendItems; e++) {
            const uint32_t i = i0 + e * blockDim.x + tid;
            if (i >= n) break;
            const Item it = item_of(i);
            const TP* p = x + (size_t)it.head * dim;
            load8(p + it.lo, u[e]);
            load8(p + (it.turn ? it.lo + half : it.lo + 8), v[e]);
        }
    };
    if constexpr (VEC) ask(0);
    const uint32_t s = sequence_of(c, row);
    if (s >= c.n_seqs) return;
    const Seq q = sequence(c, s);
    const uint32_t back = q.row0 + q.n - row;                    // rows up to the sequence's end, this one included
    // By the length as it stands there: by one that is cut to the table, rows would move onto positions that others have.
    const uint32_t pos = (uint32_t)q.given - back;
    if (row < q.row0 || row >= q.row0 + q.n || back > q.len || (q.given != (int32_t)q.len && pos >= c.table_ld << c.page_log2)) {
        report(c);                                               // starts that do not rise, more rows than positions, or a position behind the table
        return;
    }
    bool ok;
    const size_t at = page_row(c, c.table + (pos < c.shared ? 0 : (size_t)s * c.table_ld), pos, 0, &ok);      // shared positions: in the first sequence's pages
    TC *kc = reinterpret_cast<TC*>(c.k) + at, *vc = reinterpret_cast<TC*>(c.v) + at, *qo = reinterpret_cast<TC*>(a.q_out) + (size_t)row * a.ldq;
    const size_t head_stride = (size_t)dim << c.page_log2;
    // where head i of the row goes; null: nowhere
    auto target = [&](uint32_t i) -> TC* {
        if (i < c.heads) return a.q_out ? qo + (size_t)i * dim : nullptr;
        if (!ok) return nullptr;
        i -= c.heads;
        return i < c.kv_heads ? kc + i * head_stride : vc + (i - c.kv_heads) * head_stride;
    };
    if (tid < half) {
        if (pos < 1u << 17) ls::sincos_at(pos, a.freq[tid], a.freq[half + tid], &sn[tid], &cs[tid]);
        else {
            const float2 t = sincos_far(pos, a.freq[tid], a.freq[half + tid]);
            sn[tid] = t.x;
            cs[tid] = t.y;
        }
    }
    __syncthreads();
    if constexpr (VEC) {
        for (uint32_t i0 = 0; i0 < n; i0 += blockDim.x * kAppendItems) {
            if (i0 > 0) ask(i0);
#pragma unroll
            for (uint32_t e = 0; e < kAppendItems; e++) {
                const uint32_t i = i0 + e * blockDim.x + tid;
                if (i >= n) break;
                const Item it = item_of(i);
                TC* t = target(it.head);
                if (!t) continue;
                if (it.turn) {
                    float y[8], z[8];
#pragma unroll
                    for (uint32_t j = 0; j < 8; j++) {
                        const float co = cs[it.lo + j], si = sn[it.lo + j];
                        y[j] = fmaf(u[e][j], co, -(v[e][j] * si));
                        z[j] = fmaf(u[e][j], si, v[e][j] * co);
                    }
                    store8(t + it.lo, y);
                    store8(t + it.lo + half, z);
                } else {
                    store8(t + it.lo, u[e]);
                    store8(t + it.lo + 8, v[e]);
                }
            }
        }
    } else {
        const uint32_t per = dim / 2, n = (all - first) * per;
        for (uint32_t i = tid; i < n; i += blockDim.x) {
            const uint32_t head = first + i / per, d = i % per;
            TC* t = target(head);
            if (!t) continue;
            const TP* p = x + (size_t)head * dim;
            const bool turn = head < turned && d < half;
            const uint32_t lo = turn ? d : head < turned ? a.rot + 2 * (d - half) : 2 * d, hi = turn ? lo + half : lo + 1;
            const float u = to_f32(p[lo]), v = to_f32(p[hi]);
            const float co = turn ? cs[lo] : 1.f, si = turn ? sn[lo] : 0.f;
            t[lo] = from_f32<TC>(turn ? fmaf(u, co, -(v * si)) : u);
            t[hi] = from_f32<TC>(turn ? fmaf(u, si, v * co) : v);
        }
    }
}

// As many threads as a row has work for, a multiple of a warp, and one for each angle at least (8000 rows of 14 + 4 heads of 64 from f32: 96 threads 11.8 us, 192 19.9).
template <typename TP, typename TC> static void launch_append(runit_ctx* ctx, const AppendArgs& a, bool vec) {
    const uint32_t n = ((a.q_out ? a.c.heads : 0) + 2 * a.c.kv_heads) * a.c.dim / 16, threads = min(kAppendThreads, max(64u, (n / kAppendItems + 31) & ~31u));
    if (vec) runit_launch_chain(ctx, paged_append_kernel<TP, TC, true>, dim3(a.c.rows), dim3(threads), a);
    else runit_launch_chain(ctx, paged_append_kernel<TP, TC, false>, dim3(a.c.rows), dim3(kAppendThreads), a);
}

}  // namespace pg
}  // namespace runit

using namespace runit;

extern "C" int32_t runit_paged_append(runit_ctx_t* ctx, const runit_paged_cfg* cfg, const runit_paged_batch* batch, const void* proj, int32_t proj_type,
                                      uint32_t ld, const void* freq, uint32_t rot_dims, void* q_out, uint32_t ldq) {
    if (!ctx) return RUNIT_ERR_BAD_ARG;
    const char* why = pg::why_not(cfg, batch);
    if (!why) why = pg::why_not_memory(cfg, batch);
    RUNIT_REQUIRE(ctx, !why, "paged_append: %s", why);
    RUNIT_REQUIRE(ctx, proj && (proj_type == RUNIT_TYPE_F32 || proj_type == cfg->type), "paged_append: proj must be f32 or of the cache's type");
    RUNIT_REQUIRE(ctx, runit_aligned(proj, proj_type == RUNIT_TYPE_F32 ? 4 : 2) && runit_aligned(q_out, 2) && runit_aligned(freq, 4), "paged_append: misaligned proj, q_out or freq");
    RUNIT_REQUIRE(ctx, ld >= (uint64_t)(cfg->heads + 2ull * cfg->kv_heads) * cfg->dim, "paged_append: ld=%u is less than a projected row", ld);
    RUNIT_REQUIRE(ctx, !q_out || ldq >= (uint64_t)cfg->heads * cfg->dim, "paged_append: ldq=%u is less than a row of queries", ldq);
    RUNIT_REQUIRE(ctx, rot_dims % 2 == 0 && rot_dims <= cfg->dim && (freq || rot_dims == 0), "paged_append: rot_dims=%u must be even and at most dim, with frequencies", rot_dims);
    const pg::AppendArgs a{pg::cache_of(ctx, cfg, batch), proj, q_out, (const float*)freq, ld, ldq, rot_dims};
    const bool f32 = proj_type == RUNIT_TYPE_F32;
    const bool vec = rot_dims % 16 == 0 && runit_aligned(proj, 16) && ld % (f32 ? 4 : 8) == 0 && (!q_out || (runit_aligned(q_out, 16) && ldq % 8 == 0));
    if (cfg->type == RUNIT_TYPE_F16) {
        if (f32) pg::launch_append<float, __half>(ctx, a, vec);
        else pg::launch_append<__half, __half>(ctx, a, vec);
    } else {
        if (f32) pg::launch_append<float, __nv_bfloat16>(ctx, a, vec);
        else pg::launch_append<__nv_bfloat16, __nv_bfloat16>(ctx, a, vec);
    }
    return runit_after_launch(ctx, "paged_append");
}
