// Log probabilities of given tokens, entropy and the most probable entries of rows of logits.
//
// With m = max x, d = x - m, Z = sum e^d: log p = d - log Z, entropy = log Z - (sum e^d d) / Z.  The maximal entry's own 1 is kept out of the sum, Z = 1 + z
// and log Z = log1p(z): when that entry holds nearly all of the mass, its log probability and the entropy are tiny and keep their digits.
#include "gemv_common.cuh"
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

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f, kLeast = -200.f;      // e^-200 is 0 in f32

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float exp_of(float d) { return exp2_approx(d * kLog2e); }
// Order of the logits as integers: NaN before everything, one zero; 0 is below every logit.
__device__ __forceinline__ uint32_t order(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o); }

// Sums over some of a row: its maximum m; z = sum e^(x - m) and b = sum e^(x - m) (x - m) without one entry that is m.  Empty: m = -Inf.
struct Sums {
    float m, z, b;
};
// of all lanes (or as many of them as have any)
__device__ __forceinline__ Sums over_lanes(const Sums& s) {
    Sums r;
    r.m = s.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.m = max_nan(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
    const uint32_t first = __ffs(__ballot_sync(0xffffffffu, s.m == r.m)) - 1;
    const float d = s.m == -INFINITY ? kLeast : s.m - r.m, w = s.m == -INFINITY ? 0.f : exp_of(d), z = (threadIdx.x & 31) == first ? s.z : s.z + 1.f;
    r.z = w * z;
    r.b = w * fmaf(d, z, s.b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        r.z += __shfl_xor_sync(0xffffffffu, r.z, o);
        r.b += __shfl_xor_sync(0xffffffffu, r.b, o);
    }
    return r;
}

// The most probable entries seen by a warp, in descending order: lane i has the i-th.  (order of the value, ~index): equal values by index.
struct Top {
    uint32_t v, i;
};
__device__ __forceinline__ bool before(const Top& a, uint32_t v, uint32_t i) { return a.v > v || (a.v == v && a.i > i); }
__device__ __forceinline__ void insert(Top& t, uint32_t v, uint32_t i) {
    const uint32_t lane = threadIdx.x & 31, at = __popc(__ballot_sync(0xffffffffu, before(t, v, i)));
    const uint32_t uv = __shfl_up_sync(0xffffffffu, t.v, 1), ui = __shfl_up_sync(0xffffffffu, t.i, 1);
    if (lane == at) { t.v = v; t.i = i; }
    else if (lane > at) { t.v = uv; t.i = ui; }
}
// The first 32 of two such lists: the larger of one and the other from its end is a list that rises and falls, which five exchanges put in order.
__device__ __forceinline__ void join(Top& t, const Top& o) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t ov = __shfl_sync(0xffffffffu, o.v, 31 - lane), oi = __shfl_sync(0xffffffffu, o.i, 31 - lane);
    if (!before(t, ov, oi)) { t.v = ov; t.i = oi; }
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1) {
        const uint32_t xv = __shfl_xor_sync(0xffffffffu, t.v, d), xi = __shfl_xor_sync(0xffffffffu, t.i, d);
        if (before(t, xv, xi) == ((lane & d) != 0)) { t.v = xv; t.i = xi; }
    }
}

template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr uint32_t N = 4;
    static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[4]) {
        v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    }
};
template <> struct Vec<__half> {
    static constexpr uint32_t N = 8;
    static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[8]) {
        const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr uint32_t N = 8;
    static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};

// A warp's pass over its share of a row, in the order of the indices.  The maximum is the warp's: it rises some ten times in a share, and then
// only the sums are scaled; one lane leaves the maximal entry out.
template <bool TOP, int N> struct Pass {
    float m = -INFINITY;
    uint32_t owner = 32;                       // the lane that has left an entry out
    uint64_t z2 = 0, b2 = 0;
    Top top = {0, 0};
    float least = NAN;                         // the k-th so far: nothing is known of what is not above it.  NaN: fewer than k
    uint32_t k;

    __device__ __forceinline__ explicit Pass(uint32_t k_) : k(k_) {}
    // entries i, i + 1, ...: `count` of them, the others of v are -Inf
    __device__ __forceinline__ void take(const float (&v)[N], uint32_t i, uint32_t count) {
        float most = v[0];
#pragma unroll
        for (int e = 1; e < N; e++) most = max_nan(most, v[e]);
        bool leave = false;
        if (__any_sync(0xffffffffu, !(most <= m))) {
            float now = max_nan(m, most);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) now = max_nan(now, __shfl_xor_sync(0xffffffffu, now, o));
            const uint32_t lane = threadIdx.x & 31;
            const float d = m == -INFINITY ? kLeast : m - now, w = m == -INFINITY ? 0.f : exp_of(d);
            float z = sum2(z2), b = sum2(b2);
            if (lane == owner) z += 1.f;       // what was left out so far
            b = w * fmaf(d, z, b);
            z2 = pack2(__float_as_uint(w * z), 0);
            b2 = pack2(__float_as_uint(b), 0);
            m = now;
            owner = __ffs(__ballot_sync(0xffffffffu, most == now)) - 1;
            leave = lane == owner;
        }
        const float sub = m == -INFINITY ? 0.f : m;
        const uint64_t sub2 = packf(-sub), l2 = packf(kLog2e);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            uint64_t d = fadd2(pack2(__float_as_uint(v[e]), __float_as_uint(v[e + 1])), sub2);
            d = pack2(__float_as_uint(fmaxf(__uint_as_float((uint32_t)d), kLeast)), __float_as_uint(fmaxf(__uint_as_float((uint32_t)(d >> 32)), kLeast)));
            const uint64_t t = fmul2(d, l2);
            float p0 = exp2_approx(__uint_as_float((uint32_t)t)), p1 = exp2_approx(__uint_as_float((uint32_t)(t >> 32)));
            if (leave && v[e] == m) { p0 = 0.f; leave = false; }
            if (leave && v[e + 1] == m) { p1 = 0.f; leave = false; }
            const uint64_t p = pack2(__float_as_uint(p0), __float_as_uint(p1));
            z2 = fadd2(z2, p);
            b2 = ffma2(p, d, b2);
        }
        if constexpr (TOP) {
            bool open = count > 0;
            uint32_t who;
            while ((who = __ballot_sync(0xffffffffu, open && !(most <= least))) != 0) {
                const uint32_t from = __ffs(who) - 1, n = __shfl_sync(0xffffffffu, count, from), i0 = __shfl_sync(0xffffffffu, i, from);
                open = open && (threadIdx.x & 31) != from;
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float x = __shfl_sync(0xffffffffu, v[e], from);
                    if ((uint32_t)e >= n || x <= least) continue;
                    insert(top, order(x), ~(i0 + e));
                    const uint32_t last = __shfl_sync(0xffffffffu, top.v, k - 1);
                    least = last ? value(last) : NAN;
                }
            }
        }
    }
    __device__ __forceinline__ Sums sums() const {
        Sums s{m, sum2(z2), sum2(b2)};
        float z = s.z, b = s.b;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            z += __shfl_xor_sync(0xffffffffu, z, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        s.z = z;
        s.b = b;
        return s;
    }
};

// A cluster of `cluster` blocks per row (a power of two up to 16), each with a run of the row; the first one adds up.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const Args a, const uint32_t cluster) {
    constexpr uint32_t N = Vec<T>::N, kAhead = 4;
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ Sums part[kWarps], all;
    __shared__ Top tops[kWarps][32], best[32];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x / cluster, rank = blockIdx.x % cluster;
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.ld;
    // entries ahead of the first 16-byte boundary, whole vectors, entries behind the last
    const uint32_t head = min(a.n, (uint32_t)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T))), vecs = (a.n - head) / N, tail = a.n - head - vecs * N;
    const uint32_t per = (vecs + cluster - 1) / cluster, v0 = min(vecs, rank * per), v1 = min(vecs, v0 + per);
    const uint4* const xv = reinterpret_cast<const uint4*>(x + head);
    int32_t token = 0;
    float xt = 0.f;
    if (rank == 0 && tid == 0 && a.tokens) {
        token = a.tokens[row];
        if ((uint32_t)token < a.n) xt = to_f32(x[token]);
    }
    Pass<TOP, N> pass(a.k);
    float v[N];
    auto few = [&](uint32_t first, uint32_t count) {             // up to N - 1 entries, one a lane
#pragma unroll
        for (uint32_t e = 0; e < N; e++) v[e] = -INFINITY;
        if (lane < count) v[0] = to_f32(x[first + lane]);
        pass.take(v, first + lane, lane < count ? 1 : 0);
    };
    if (rank == 0 && warp == 0 && head) few(0, head);
    uint32_t i = v0 + tid;
    for (; i - tid + kThreads * kAhead <= v1; i += kThreads * kAhead) {
        uint4 u[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++) u[j] = __ldcs(xv + i + j * kThreads);
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++) {
            Vec<T>::unpack(u[j], v);
            pass.take(v, head + (i + j * kThreads) * N, N);
        }
    }
    for (; i - lane < v1; i += kThreads) {
        const bool in = i < v1;
        if (in) Vec<T>::unpack(__ldcs(xv + i), v);
        else {
#pragma unroll
            for (uint32_t e = 0; e < N; e++) v[e] = -INFINITY;
        }
        pass.take(v, head + i * N, in ? N : 0);
    }
    if (rank == cluster - 1 && warp == kWarps - 1 && tail) few(head + vecs * N, tail);
    const Sums mine = pass.sums();
    if (lane == 0) part[warp] = mine;
    if (TOP) tops[warp][lane] = pass.top;
    __syncthreads();
    Top t = {0, 0};
    if (warp == 0) {
        const Sums s = over_lanes(lane < kWarps ? part[lane] : Sums{-INFINITY, 0.f, 0.f});
        if (lane == 0) all = s;
        if (TOP) {
            t = pass.top;
            for (uint32_t w = 1; w < kWarps; w++) join(t, tops[w][lane]);
            best[lane] = t;
        }
    }
    __syncwarp();
    if (cluster > 1) cluster_sync();
    if (rank == 0 && warp == 0) {
        Sums s{-INFINITY, 0.f, 0.f};
        if (lane < cluster) s = Sums{ld_cluster_f32(&all.m, lane), ld_cluster_f32(&all.z, lane), ld_cluster_f32(&all.b, lane)};
        s = over_lanes(s);
        if (TOP)
            for (uint32_t w = 1; w < cluster; w++)
                join(t, Top{__float_as_uint(ld_cluster_f32(reinterpret_cast<const float*>(&best[lane].v), w)), __float_as_uint(ld_cluster_f32(reinterpret_cast<const float*>(&best[lane].i), w))});
        const bool none = s.m == -INFINITY;
        if (s.m == INFINITY) s.z = NAN;        // Inf - Inf, as the formula has it
        const float logz = log1pf(s.z);
        auto log_of = [&](float y) { return y == -INFINITY && s.m == s.m && s.z == s.z ? -INFINITY : y - s.m - logz; };
        if (lane == 0) {
            if (a.entropy) a.entropy[row] = none ? 0.f : s.m == s.m ? logz - s.b / (1.f + s.z) : NAN;
            if (a.tokens) a.logprob[row] = (uint32_t)token < a.n ? log_of(xt) : 0.f;
        }
        if (TOP && lane < a.k) {
            a.top_ids[(size_t)row * a.k + lane] = (int32_t)~t.i;
            a.top_logprobs[(size_t)row * a.k + lane] = log_of(value(t.v));
        }
    }
    __syncwarp();
    if (cluster > 1) cluster_sync();           // the others' sums are read by then
}

// Blocks of a row: enough rows fill the GPU by themselves; a block has 2048 entries at least.
static uint32_t cluster_of(uint32_t rows, uint32_t n) {
    uint32_t c = 1;
    while (c < 16 && (uint64_t)rows * c * 2 <= 2 * 148 && n / (c * 2) >= 2048) c *= 2;
    return c;
}
template <typename T, bool TOP> static int32_t run(runit_ctx* ctx, const Args& a, uint32_t rows) {
    const uint32_t cluster = cluster_of(rows, a.n);
    static bool configured[64] = {false};
    if (ctx->device >= 64 || !configured[ctx->device]) {
        RUNIT_CUDA_TRY(ctx, cudaFuncSetAttribute(token_logprobs_kernel<T, TOP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (ctx->device < 64) configured[ctx->device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * cluster);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->tune.pdl != 0 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, TOP>, a, cluster);           // errors surface in runit_after_launch
    return runit_after_launch(ctx, "token_logprobs");
}

}  // namespace lp
}  // namespace runit

using namespace runit;

extern "C" int32_t runit_token_logprobs(runit_ctx_t* ctx, const void* logits, int32_t type, uint32_t ld, uint32_t n, uint32_t rows, const void* tokens,
                                        void* logprob, void* entropy, uint32_t k, void* top_ids, void* top_logprobs) {
    if (!ctx) return RUNIT_ERR_BAD_ARG;
    RUNIT_REQUIRE(ctx, type >= RUNIT_TYPE_F32 && type <= RUNIT_TYPE_BF16, "token_logprobs: type %d", type);
    RUNIT_REQUIRE(ctx, logits && n > 0 && rows > 0 && ld >= n && n <= 0x7FFFFFFFu && rows <= 0x7FFFFFFFu / 16, "token_logprobs: null logits, n=%u, rows=%u or ld=%u", n, rows, ld);
    RUNIT_REQUIRE(ctx, runit_aligned(logits, type == RUNIT_TYPE_F32 ? 4 : 2), "token_logprobs: misaligned logits");
    RUNIT_REQUIRE(ctx, (tokens != nullptr) == (logprob != nullptr), "token_logprobs: tokens and logprob come together");
    RUNIT_REQUIRE(ctx, k <= 32 && k <= n && (k > 0) == (top_ids != nullptr) && (k > 0) == (top_logprobs != nullptr), "token_logprobs: k=%u must be at most 32 and n, with top_ids and top_logprobs", k);
    RUNIT_REQUIRE(ctx, logprob || entropy || k > 0, "token_logprobs: nothing is asked for");
    RUNIT_REQUIRE(ctx, runit_aligned(tokens, 4) && runit_aligned(logprob, 4) && runit_aligned(entropy, 4) && runit_aligned(top_ids, 4) && runit_aligned(top_logprobs, 4),
                  "token_logprobs: misaligned tokens or results");
    const lp::Args a{logits, (const int32_t*)tokens, (float*)logprob, (float*)entropy, (float*)top_logprobs, (int32_t*)top_ids, ld, n, k};
    if (type == RUNIT_TYPE_F32) return k ? lp::run<float, true>(ctx, a, rows) : lp::run<float, false>(ctx, a, rows);
    if (type == RUNIT_TYPE_F16) return k ? lp::run<__half, true>(ctx, a, rows) : lp::run<__half, false>(ctx, a, rows);
    return k ? lp::run<__nv_bfloat16, true>(ctx, a, rows) : lp::run<__nv_bfloat16, false>(ctx, a, rows);
}
