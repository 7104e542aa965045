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

constexpr float kFloor = -1e38f;               // -Inf in the fast path, where the maximum is above kLow, so far above that the floor has no mass

// Sixteen bytes of logits: unpacked; their maximum (a NaN stays one); unpacked with -Inf raised to the floor (f16: to its lowest number).
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr uint32_t N = 4;
    static constexpr float kLow = -1e37f;
    static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[4]) {
        v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ float most(const uint4& u) {
        return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)), max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
    }
    static __device__ __forceinline__ void raised(const uint4& u, float (&v)[4]) {
        unpack(u, v);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = fmaxf(v[i], kFloor);
    }
    static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u); }
    static __device__ __forceinline__ uint4 one(float v) { return make_uint4(__float_as_uint(v), 0xFF800000u, 0xFF800000u, 0xFF800000u); }
};
template <> struct Vec<__half> {
    static constexpr uint32_t N = 8;
    static constexpr float kLow = -6e4f;
    static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[8]) {
        const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ float most(const uint4& u) {
        const __half2* h = reinterpret_cast<const __half2*>(&u);
        const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return max_nan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ void raised(const uint4& u, float (&v)[8]) {
        uint4 r;
        const __half2 low = __half2half2(__ushort_as_half(0xFBFF));
#pragma unroll
        for (int i = 0; i < 4; i++) reinterpret_cast<__half2*>(&r)[i] = __hmax2(reinterpret_cast<const __half2*>(&u)[i], low);
        unpack(r, v);
    }
    static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u); }
    static __device__ __forceinline__ uint4 one(__half v) { return make_uint4(0xFC000000u | __half_as_ushort(v), 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u); }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr uint32_t N = 8;
    static constexpr float kLow = -1e37f;
    static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ float most(const uint4& u) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return max_nan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ void raised(const uint4& u, float (&v)[8]) {
        uint4 r;
        const __nv_bfloat162 low = __bfloat162bfloat162(__ushort_as_bfloat16(0xFE96));           // -1e38
#pragma unroll
        for (int i = 0; i < 4; i++) reinterpret_cast<__nv_bfloat162*>(&r)[i] = __hmax2(reinterpret_cast<const __nv_bfloat162*>(&u)[i], low);
        unpack(r, v);
    }
    static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }
    static __device__ __forceinline__ uint4 one(__nv_bfloat16 v) { return make_uint4(0xFF800000u | __bfloat16_as_ushort(v), 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }
};

// A warp's pass over its share of a row, in the order of the indices.  The maximum is the warp's: it rises some ten times in a share, and only
// then are the sums scaled; one lane leaves the maximal entry out.
template <typename T, bool TOP> struct Pass {
    static constexpr uint32_t N = Vec<T>::N;
    float m = -INFINITY, mine = -INFINITY;     // of the warp; of the lane's vectors
    uint32_t owner = 32, at = 0xFFFFFFFFu;     // the lane that has left an entry out; the lane's first vector that has `mine`
    uint64_t z2 = 0, b2 = 0;

    // vector i of the row (-Inf where there is nothing; `in`: it counts among the lane's)
    __device__ __forceinline__ void take(const uint4& u, uint32_t i, bool in) {
        const float most = Vec<T>::most(u);
        const bool up = !(most <= m);
        if (__any_sync(0xffffffffu, up || m < Vec<T>::kLow)) {
            rise(u, most, i, in);
            return;
        }
        if (TOP && most > mine && in) { mine = most; at = i; }
        float v[N];
        Vec<T>::raised(u, v);
        const uint64_t sub2 = packf(-m), l2 = packf(kLog2e);
#pragma unroll
        for (uint32_t e = 0; e < N; e += 2) {
            const uint64_t d = fadd2(pack2(__float_as_uint(v[e]), __float_as_uint(v[e + 1])), sub2), t = fmul2(d, l2);
            const uint64_t p = pack2(__float_as_uint(exp2_approx(__uint_as_float((uint32_t)t))), __float_as_uint(exp2_approx(__uint_as_float((uint32_t)(t >> 32)))));
            z2 = fadd2(z2, p);
            b2 = ffma2(p, d, b2);
        }
    }
    // the same where the maximum rises, is no number or is very low
    __device__ __forceinline__ void rise(const uint4& u, float most, uint32_t i, bool in) {
        const uint32_t lane = threadIdx.x & 31;
        if (TOP && in && (most > mine || (most != most && mine == mine))) { mine = most; at = i; }
        bool leave = false;
        if (__any_sync(0xffffffffu, !(most <= m))) {
            float now = max_nan(m, most);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) now = max_nan(now, __shfl_xor_sync(0xffffffffu, now, o));
            const float d = m == -INFINITY ? kLeast : m - now, w = m == -INFINITY ? 0.f : exp_of(d);
            const float z = sum2(z2) + (lane == owner ? 1.f : 0.f), b = sum2(b2);         // with what was left out so far
            z2 = pack2(__float_as_uint(w * z), 0);
            b2 = pack2(__float_as_uint(w * fmaf(d, z, b)), 0);
            m = now;
            owner = __ffs(__ballot_sync(0xffffffffu, most == now)) - 1;
            leave = lane == owner;
        }
        const float sub = m == -INFINITY ? 0.f : m;
        float v[N], z = 0.f, b = 0.f;
        Vec<T>::unpack(u, v);
#pragma unroll
        for (uint32_t e = 0; e < N; e++) {
            const float d = fmaxf(v[e] - sub, kLeast);
            float p = exp_of(d);
            if (leave && v[e] == m) { p = 0.f; leave = false; }
            z += p;
            b = fmaf(p, d, b);
        }
        z2 = fadd2(z2, pack2(__float_as_uint(z), 0));
        b2 = fadd2(b2, pack2(__float_as_uint(b), 0));
    }
    // the lane's largest entry; first: its first vector, if it has any
    __device__ __forceinline__ Top top(uint32_t first, uint32_t end) const {
        if (at != 0xFFFFFFFFu) return Top{order(mine), ~at};
        return first < end ? Top{order(-INFINITY), ~first} : Top{0, 0};
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

// The lists of a block's warps joined: the result in warp 0.  All threads.
__device__ __forceinline__ void join_warps(Top& t, Top (*lists)[32]) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    lists[warp][lane] = t;
    __syncthreads();
#pragma unroll
    for (uint32_t w = kWarps / 2; w > 0; w /= 2) {
        if (warp < w) {
            join(t, lists[warp + w][lane]);
            lists[warp][lane] = t;
        }
        __syncthreads();
    }
}
// Descending order of the lanes' entries.
__device__ __forceinline__ void sort_lanes(Top& t) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (uint32_t n = 2; n <= 32; n *= 2)
#pragma unroll
        for (uint32_t d = n / 2; d > 0; d /= 2) {
            const uint32_t xv = __shfl_xor_sync(0xffffffffu, t.v, d), xi = __shfl_xor_sync(0xffffffffu, t.i, d);
            const bool up = (lane & n) != 0;                     // this stretch ascends
            if (before(t, xv, xi) == (((lane & d) != 0) != up) && (t.v != xv || t.i != xi)) { t.v = xv; t.i = xi; }
        }
}

// A cluster of `cluster` blocks per row (a power of two up to 16), each with a run of the row; the first one adds up.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const Args a, const uint32_t cluster) {
    constexpr uint32_t N = Vec<T>::N, kAhead = 4;
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ Sums part[kWarps], all;
    __shared__ Top lists[kWarps][32], best[32];
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
    Pass<T, TOP> pass;
    // up to N - 1 entries, one a lane
    auto few = [&](uint32_t first, uint32_t count) { pass.take(lane < count ? Vec<T>::one(x[first + lane]) : Vec<T>::nothing(), 0, false); };
    if (rank == 0 && warp == 0 && head) few(0, head);
    uint32_t i = v0 + tid;
    for (; i - tid + kThreads * kAhead <= v1; i += kThreads * kAhead) {
        uint4 u[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++) u[j] = __ldcs(xv + i + j * kThreads);
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++) pass.take(u[j], i + j * kThreads, true);
    }
    {
        uint4 u[kAhead];                       // what is left: all requested before the first is looked at
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++) u[j] = i + j * kThreads < v1 ? __ldcs(xv + i + j * kThreads) : Vec<T>::nothing();
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++)
            if (i - lane + j * kThreads < v1) pass.take(u[j], i + j * kThreads, i + j * kThreads < v1);
    }
    if (rank == cluster - 1 && warp == kWarps - 1 && tail) few(head + vecs * N, tail);
    const Sums mine = pass.sums();
    if (lane == 0) part[warp] = mine;
    Top t = {0, 0};
    if constexpr (TOP) {
        // The k lanes with the largest entries have the k largest entries of all among theirs, whatever is larger than the k-th lane's: only those lanes' vectors
        // are looked at again.  (Order by value, then by vector: of equal values in one vector all are taken.)
        t = pass.top(v0 + tid, v1);
        sort_lanes(t);
        join_warps(t, lists);
        const Top least = lists[0][a.k - 1];
        Top found = {0, 0};
        auto offer = [&](float y, uint32_t vec, uint32_t id, bool in) {      // entry `id` of a lane's vector `vec`
            const uint32_t o = order(y);
            uint32_t who = __ballot_sync(0xffffffffu, in && (o > least.v || (o == least.v && ~vec >= least.i)));
            while (who) {
                const uint32_t from = __ffs(who) - 1;
                who &= who - 1;
                insert(found, __shfl_sync(0xffffffffu, o, from), __shfl_sync(0xffffffffu, ~id, from));
            }
        };
        uint32_t wide = 1;                     // threads of this warp that look at one lane's vectors: as many as it has, if that is fewer than 32
        while (wide < 32 && wide * kThreads < v1 - v0) wide *= 2;
        for (uint32_t q0 = warp * (32 / wide); q0 < a.k; q0 += kThreads / wide) {
            const uint32_t q = q0 + lane / wide;
            const Top s = q < a.k ? lists[0][q] : Top{0, 0};
            const uint32_t first = s.v ? v0 + (~s.i - v0) % kThreads + lane % wide * kThreads : v1;
            for (uint32_t j = 0; __any_sync(0xffffffffu, first + j < v1); j += kThreads * wide) {
                const bool in = first + j < v1;
                float v[N];
                Vec<T>::unpack(in ? xv[first + j] : Vec<T>::nothing(), v);
#pragma unroll
                for (uint32_t e = 0; e < N; e++) offer(v[e], first + j, head + (first + j) * N + e, in);
            }
        }
        // the entries outside of the vectors: those in front come before all others of their value, those behind after them
        if (rank == 0 && warp == 0 && head) offer(lane < head ? to_f32(x[lane]) : 0.f, 0, lane, lane < head);
        if (rank == cluster - 1 && warp == kWarps - 1 && tail) {
            const uint32_t id = head + vecs * N + lane;
            offer(lane < tail ? to_f32(x[id]) : 0.f, vecs, id, lane < tail);
        }
        __syncthreads();                       // `least` and the lanes have been read
        t = found;
        join_warps(t, lists);
        if (warp == 0) best[lane] = t;
    }
    __syncthreads();
    if (warp == 0) {
        const Sums s = over_lanes(lane < kWarps ? part[lane] : Sums{-INFINITY, 0.f, 0.f});
        if (lane == 0) all = s;
    }
    __syncwarp();
    if (cluster > 1) cluster_sync();
    if (TOP && rank == 0 && cluster > 1) {     // a warp per block, or two
        t = {0, 0};
        for (uint32_t w = warp; w < cluster; w += kWarps)
            join(t, Top{__float_as_uint(ld_cluster_f32(reinterpret_cast<const float*>(&best[lane].v), w)), __float_as_uint(ld_cluster_f32(reinterpret_cast<const float*>(&best[lane].i), w))});
        join_warps(t, lists);
    }
    if (rank == 0 && warp == 0) {
        Sums s{-INFINITY, 0.f, 0.f};
        if (lane < cluster) s = Sums{ld_cluster_f32(&all.m, lane), ld_cluster_f32(&all.z, lane), ld_cluster_f32(&all.b, lane)};
        s = over_lanes(s);
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
