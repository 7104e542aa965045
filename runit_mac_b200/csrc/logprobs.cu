// Log probabilities of given tokens, entropy and the most probable entries of rows of logits.
//
// With m = max x, d = x - m, Z = sum e^d: log p = d - log Z, entropy = log Z - (sum e^d d) / Z.  The maximal entry's own 1 is kept out of the sum, Z = 1 + z
// and log Z = log1p(z): when that entry holds nearly all of the mass, its log probability and the entropy are tiny and keep their digits.
// Bound: HBM and the issue slots, close to each other: 2048 rows of 152064 bf16 logits with 5 alternatives take 123 to 131 us, 5.1 to 4.8 TB/s
// (three GPUs).  Few rows: latency; 8 rows of 151936 with 20 alternatives, a cluster of 16 blocks for each, 13.2 us.
#include "gemv_common.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace runit {
namespace lp {

using pg::to_f32;

struct Args {
    const void* x;
    const int32_t* tokens;
    float *logprob, *entropy, *top_logprobs;
    int32_t* top_ids;
    int32_t* status;
    uint32_t ld, n, k, rows;
};

constexpr uint32_t kWarps = 7, kAhead = 4, kStages = 3;     // kWarps read; one or two more add up what they have found
constexpr uint32_t kStageVecs = 32 * kAhead, kStageBytes = 16 * kStageVecs, kBlocksPerSm = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kLeast = -200.f;      // e^-200 is 0 in f32

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
// The k largest entries of those that the lanes have at key(0) (a lane's next one comes up when next() is called in it), in descending order over the lanes.
template <typename Key, typename Next> __device__ __forceinline__ Top largest(uint32_t k, Key key, Next next) {
    const uint32_t lane = threadIdx.x & 31;
    Top t = {0, 0};
#pragma unroll 1
    for (uint32_t j = 0; j < k; j++) {
        const Top mine = key();
        const uint32_t v = __reduce_max_sync(0xffffffffu, mine.v);
        if (v == 0) break;
        uint32_t who = __ballot_sync(0xffffffffu, mine.v == v);
        if (who & (who - 1)) {                 // equal ones: the lowest index
            const uint32_t i = __reduce_max_sync(0xffffffffu, mine.v == v ? mine.i : 0);
            who = __ballot_sync(0xffffffffu, mine.v == v && mine.i == i);
        }
        const uint32_t from = __ffs(who) - 1, i = __shfl_sync(0xffffffffu, mine.i, from);
        if (lane == j) { t.v = v; t.i = i; }
        if (lane == from) next();
    }
    return t;
}

constexpr float kFloor = -1e38f;               // -Inf in the fast path, where the maximum is within kFar: far above the floor, and R is rounded by less than 2^-7

// Sixteen bytes of logits: unpacked; their maximum (a NaN stays one); unpacked with -Inf raised to the floor (f16: to its lowest number).
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr uint32_t N = 4;
    static constexpr float kFar = 1e5f;
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
    // the first entry that is m becomes -Inf
    static __device__ __forceinline__ void drop(uint4& u, float m, bool& leave) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (leave && __uint_as_float(w[i]) == m) { w[i] = 0xFF800000u; leave = false; }
    }
    static __device__ __forceinline__ uint4 one(float v) { return make_uint4(__float_as_uint(v), 0xFF800000u, 0xFF800000u, 0xFF800000u); }
};
template <> struct Vec<__half> {
    static constexpr uint32_t N = 8;
    static constexpr float kFar = 6e4f;
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
    static __device__ __forceinline__ void drop(uint4& u, float m, bool& leave) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int q = 0; q < 2; q++)
                if (leave && __half2float(__ushort_as_half((unsigned short)(w[i] >> 16 * q))) == m) {
                    w[i] = (w[i] & (0xFFFF0000u >> 16 * q)) | (0xFC00u << 16 * q);
                    leave = false;
                }
    }
    static __device__ __forceinline__ uint4 one(__half v) { return make_uint4(0xFC000000u | __half_as_ushort(v), 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u); }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr uint32_t N = 8;
    static constexpr float kFar = 1e5f;
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
    static __device__ __forceinline__ void drop(uint4& u, float m, bool& leave) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int q = 0; q < 2; q++)
                if (leave && __uint_as_float((w[i] >> 16 * q) << 16) == m) {
                    w[i] = (w[i] & (0xFFFF0000u >> 16 * q)) | (0xFF80u << 16 * q);
                    leave = false;
                }
    }
    static __device__ __forceinline__ uint4 one(__nv_bfloat16 v) { return make_uint4(0xFF800000u | __bfloat16_as_ushort(v), 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }
};

// A warp's pass over its share of a row, in the order of the indices.  The maximum is the warp's: it rises some five to ten times in a share, and only
// then are the sums scaled; one lane leaves the maximal entry out.  Below the maximum an entry is one multiply-add, t = x log2 e - R with R = m log2 e
// rounded, 2^t and the sums of 2^t and 2^t t; what R was rounded by (e) goes into the sums when they are handed over.
template <typename T, bool TOP> struct Pass {
    static constexpr uint32_t N = Vec<T>::N;
    float m = -INFINITY;
    uint32_t owner = 32;                       // the lane that has left an entry out
    float mine = -INFINITY, second = -INFINITY;                  // the largest entries of the lane's vectors: of one, and of the others
    uint32_t at = 0xFFFFFFFFu;                 // the first vector that has `mine`
    bool nan = false, leave = false;
    float z = 0.f, b = 0.f, r = 0.f;           // sums of e^d and e^d d relative to m; R
    uint64_t z2 = 0, b2 = 0;                   // sums of 2^t and 2^t t since m has risen

    __device__ __forceinline__ void hand_over() {
        const float e = fmaf(m, kLog2e, -r), f = exp2_approx(-e), zs = sum2(z2), bs = sum2(b2);
        if (zs != 0.f) {                       // else nothing was added (and m need not be a number)
            z = fmaf(f, zs, z);
            b = fmaf(f * kLn2, fmaf(-e, zs, bs), b);
        }
        z2 = b2 = 0;
    }
    // vectors i, i + 32, ... of the row, -Inf where there is nothing
    template <int V> __device__ __forceinline__ void take(uint4 (&u)[V], uint32_t i) {
        float most[V], all = -INFINITY;
#pragma unroll
        for (int j = 0; j < V; j++) {
            most[j] = Vec<T>::most(u[j]);
            all = max_nan(all, most[j]);
        }
        if (__any_sync(0xffffffffu, !(all <= m) || !(fabsf(m) < Vec<T>::kFar))) {
            if (!rise(all)) {                  // no number, or far out
#pragma unroll 1
                for (int j = 0; j < V; j++) {
                    uint4 x = u[0];
                    float y = most[0];
#pragma unroll
                    for (int q = 1; q < V; q++)
                        if (q == j) { x = u[q]; y = most[q]; }
                    plain(x, y, i + 32 * j);
                }
                return;
            }
            if (leave) {                       // the entry goes where the floor is
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (leave && most[j] == m) Vec<T>::drop(u[j], m, leave);
            }
        }
#pragma unroll
        for (int j = 0; j < V; j++) below(u[j], most[j], i + 32 * j);
    }
    // a vector below the maximum
    __device__ __forceinline__ void below(const uint4& u, float most, uint32_t i) {
        if (TOP) note(most, i);
        float v[N];
        Vec<T>::raised(u, v);
        const uint64_t r2 = packf(-r), l2 = packf(kLog2e);
#pragma unroll
        for (uint32_t e = 0; e < N; e += 2) {
            const uint64_t t = ffma2(pack2(__float_as_uint(v[e]), __float_as_uint(v[e + 1])), l2, r2);
            const uint64_t p = pack2(__float_as_uint(exp2_approx(__uint_as_float((uint32_t)t))), __float_as_uint(exp2_approx(__uint_as_float((uint32_t)(t >> 32)))));
            z2 = fadd2(z2, p);
            b2 = ffma2(p, t, b2);
        }
    }
    __device__ __forceinline__ void note(float most, uint32_t i) {
        second = fmaxf(second, fminf(mine, most));
        if (most > mine) { mine = most; at = i; }
    }
    // The warp's maximum becomes that of `all` too, if that is larger: the sums are scaled, one lane has an entry to leave out.  Whether 2^t can follow.
    __device__ __forceinline__ bool rise(float all) {
        const uint32_t lane = threadIdx.x & 31;
        leave = false;
        if (__any_sync(0xffffffffu, !(all <= m))) {
            float now = max_nan(m, all);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) now = max_nan(now, __shfl_xor_sync(0xffffffffu, now, o));
            hand_over();
            const float d = m == -INFINITY ? kLeast : m - now, w = m == -INFINITY ? 0.f : exp_of(d);
            if (lane == owner) z += 1.f;       // what was left out so far
            b = w * fmaf(d, z, b);
            z *= w;
            m = now;
            r = m * kLog2e;
            owner = __ffs(__ballot_sync(0xffffffffu, all == now)) - 1;
            leave = lane == owner;
        }
        return fabsf(m) < Vec<T>::kFar;
    }
    // a vector by its differences from the maximum
    __device__ __forceinline__ void plain(const uint4& u, float most, uint32_t i) {
        if (TOP) {
            if (most != most) {
                if (!nan) { mine = most; at = i; }
                nan = true;
            } else if (!nan) note(most, i);
        }
        const float sub = m == -INFINITY ? 0.f : m;
        float v[N];
        Vec<T>::unpack(u, v);
#pragma unroll
        for (uint32_t e = 0; e < N; e++) {
            const float d = fmaxf(v[e] - sub, kLeast);
            float p = exp_of(d);
            if (leave && v[e] == m) { p = 0.f; leave = false; }
            z += p;
            b = fmaf(p, d, b);
        }
    }
    // the lane's largest entry; first: its first vector, if it has any
    __device__ __forceinline__ Top top(uint32_t first, uint32_t end) const {
        if (at != 0xFFFFFFFFu) return Top{order(mine), ~at};
        return first < end ? Top{order(-INFINITY), ~first} : Top{0, 0};
    }
    // what the lane's other vectors have at most
    __device__ __forceinline__ uint32_t others() const { return nan ? 0xFFFFFFFFu : order(second); }
    __device__ __forceinline__ Sums sums() {
        hand_over();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            z += __shfl_xor_sync(0xffffffffu, z, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        return Sums{m, z, b};
    }
};

// The first k of the warps' lists, in descending order.
__device__ __forceinline__ Top first_of(const Top (&lists)[kWarps][32], uint32_t k) {
    const uint32_t lane = threadIdx.x & 31;
    Top x[kWarps];
#pragma unroll
    for (uint32_t w = 0; w < kWarps; w++) x[w] = lists[w][lane];
    auto order2 = [&](uint32_t i, uint32_t j) {
        if (before(x[i], x[j].v, x[j].i)) return;
        const Top y = x[i];
        x[i] = x[j];
        x[j] = y;
    };
    // a lane's seven, by a network of sixteen exchanges
    order2(0, 6); order2(2, 3); order2(4, 5);
    order2(0, 2); order2(1, 4); order2(3, 6);
    order2(0, 1); order2(2, 5); order2(3, 4);
    order2(1, 2); order2(4, 6);
    order2(2, 3); order2(4, 5);
    order2(1, 2); order2(3, 4); order2(5, 6);
    return largest(k, [&]() { return x[0]; }, [&]() {
#pragma unroll
        for (uint32_t w = 0; w + 1 < kWarps; w++) x[w] = x[w + 1];
        x[kWarps - 1] = Top{0, 0};
    });
}

// Counted on mbarriers, with the suspension of mbar_try: a warp that polls takes issue slots from those that have data.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < kSpinLimit; i++)
        if (mbar_try(bar, parity)) return true;
    return false;
}

// A block takes rows blockIdx.x / cluster, + gridDim.x, ...; with few rows a cluster of `cluster` blocks (a power of two up to 16) shares one, and the first of them
// adds up.  Seven warps read: the row's 16-byte vectors go to them in turn, 128 at a time, which come by a bulk copy of 2 KB into the warp's ring of three,
// and a warp goes on to the next row when it is through; the eighth warp (and a ninth, in turn)
// turns what they have found into the row's results, one row behind.
template <typename T, bool TOP, uint32_t ADDERS>
__global__ void __launch_bounds__(32 * (kWarps + ADDERS), kBlocksPerSm) token_logprobs_kernel(const Args a, const uint32_t cluster) {
    constexpr uint32_t N = Vec<T>::N;
    extern __shared__ __align__(128) uint8_t ring[];             // [kWarps][kStages][kStageBytes]
    __shared__ __align__(8) uint64_t bars[kWarps * kStages + 4];
    __shared__ Sums part[2][kWarps], blocks[16];
    __shared__ Top lists[2][kWarps][32], best[16][32];           // blocks, best: of a cluster, in its first block
    __shared__ uint32_t seconds[2][kWarps][32];
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, rank = blockIdx.x % cluster;
    if (tid < kWarps * kStages + 4) mbar_init(smem_u32(&bars[tid]), tid >= kWarps * kStages && tid < kWarps * kStages + 2 ? kWarps : 1);
    fence_mbar_init();
    if (cluster > 1) cluster_sync();           // the others run, too: their shared memory can be written
    else __syncthreads();
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t there = smem_u32(&bars[kWarps * kStages]), taken = there + 16;          // of the two buffers that hold a row's findings
    // A row: entries ahead of the first 16-byte boundary, whole vectors, entries behind the last; the block's vectors v0 .. v1 - 1.
    struct Run {
        const T* x;
        uint32_t head, vecs, tail, v0, v1;
    };
    auto run_of = [&](uint32_t row) {
        Run r;
        r.x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.ld;
        r.head = min(a.n, (uint32_t)((16 - (reinterpret_cast<uintptr_t>(r.x) & 15)) % 16 / sizeof(T)));
        r.vecs = (a.n - r.head) / N;
        r.tail = a.n - r.head - r.vecs * N;
        const uint32_t per = (r.vecs + cluster - 1) / cluster;
        r.v0 = min(r.vecs, rank * per);
        r.v1 = min(r.vecs, r.v0 + per);
        return r;
    };
    bool ok = true;
    Sums s{-INFINITY, 0.f, 0.f};               // of the warp that adds up: the block's, in the end
    Top t = {0, 0};
    uint32_t turn = 0;
    if (warp < kWarps) {
        const uint4* const mine = reinterpret_cast<const uint4*>(ring + warp * kStages * kStageBytes);
        const uint32_t mine_s = smem_u32(mine), bar0 = smem_u32(&bars[warp * kStages]);
        // The copies run ahead of the reading, on into the next row.  (What is kept here is what a copy costs least with:
        // some 80 instructions for each of them were a quarter of all.)
        uint32_t asked = 0, ask_slot = 0, slot = 0, phase = 0;
        uint32_t ask_row = blockIdx.x / cluster, left = 0;
        const uint4* next = nullptr;
        auto enter = [&]() {                   // the run of ask_row
            const Run q = run_of(ask_row);
            left = q.v1 - q.v0 > warp * kStageVecs ? q.v1 - q.v0 - warp * kStageVecs : 0;
            next = reinterpret_cast<const uint4*>(q.x + q.head) + q.v0 + warp * kStageVecs;
        };
        enter();
        auto ask = [&]() {
            while (left == 0) {
                if (cluster > 1 || a.rows - ask_row <= gridDim.x) return;
                ask_row += gridDim.x;
                enter();
            }
            const uint32_t n = min(left, kStageVecs);
            if (lane == 0) {
                mbar_expect_tx(bar0 + 8 * ask_slot, 16 * n);
                bulk_load_1d(mine_s + ask_slot * kStageBytes, next, 16 * n, bar0 + 8 * ask_slot);
            }
            asked++;
            ask_slot = ask_slot == kStages - 1 ? 0 : ask_slot + 1;
            next += kWarps * kStageVecs;
            left -= min(left, kWarps * kStageVecs);
        };
        for (uint32_t i = 0; i < kStages; i++) ask();
        for (uint32_t row = blockIdx.x / cluster;; turn++) {
            const Run r = run_of(row);
            const uint32_t w0 = r.v0 + warp * kStageVecs, w1 = r.v1, half = turn & 1;
            Pass<T, TOP> pass;
            // up to N - 1 entries, one a lane
            auto few = [&](uint32_t first, uint32_t count) {
                const uint4 u = lane < count ? Vec<T>::one(r.x[first + lane]) : Vec<T>::nothing();
                const auto was = pass;         // they do not count among the lane's vectors
                pass.rise(Vec<T>::most(u));
                pass.plain(u, Vec<T>::most(u), 0);
                pass.mine = was.mine; pass.second = was.second; pass.at = was.at; pass.nan = was.nan;
            };
            if (rank == 0 && warp == 0 && r.head) few(0, r.head);
            for (uint32_t v = w0; v < w1; v += kWarps * kStageVecs) {
                const uint4* const from = mine + slot * kStageVecs + lane;
                if (ok) ok = __all_sync(0xffffffffu, wait(bar0 + 8 * slot, phase));
                uint4 u[kAhead];
                if (v + kStageVecs <= w1) {
#pragma unroll
                    for (uint32_t j = 0; j < kAhead; j++) u[j] = from[32 * j];
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < kAhead; j++) u[j] = v + 32 * j + lane < w1 ? from[32 * j] : Vec<T>::nothing();
                }
                if (++slot == kStages) {
                    slot = 0;
                    phase ^= 1;
                }
                __syncwarp();
                if (ok) ask();
                pass.take(u, v + lane);
            }
            if (rank == cluster - 1 && warp == kWarps - 1 && r.tail) few(r.head + r.vecs * N, r.tail);
            const Sums sums = pass.sums();
            if (turn >= 2 && ok) ok = __all_sync(0xffffffffu, wait(taken + 8 * half, (turn / 2 - 1) & 1));
            if (lane == 0) part[half][warp] = sums;
            if constexpr (TOP) {
                seconds[half][warp][lane] = pass.others();
                lists[half][warp][lane] = pass.top(w0 + lane, w1);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(there + 8 * half);
            if (cluster > 1 || a.rows - row <= gridDim.x) break;
            row += gridDim.x;
        }
        if (!ok) mbar_drain(bar0, kStages, asked);               // nothing is in flight when the block leaves
    }
    bool listed = false;                       // the row's token is one of its entries, with the logit `given`
    float given = 0.f;
    auto token_of = [&](uint32_t row) {        // fetched ahead of the row's sums
        if (lane > 0 || !a.tokens) return;
        const int32_t token = a.tokens[row];
        listed = (uint32_t)token < a.n;
        if (listed) given = to_f32(reinterpret_cast<const T*>(a.x)[(size_t)row * a.ld + token]);
    };
    auto result = [&](uint32_t row) {          // of a row whose sums and alternatives are in s and t
        const bool none = s.m == -INFINITY;
        if (s.m == INFINITY) s.z = NAN;        // Inf - Inf, as the formula has it
        const float logz = log1pf(s.z);
        auto log_of = [&](float y) { return y == -INFINITY && s.m == s.m && s.z == s.z ? -INFINITY : y - s.m - logz; };
        if (lane == 0) {
            if (a.entropy) a.entropy[row] = none ? 0.f : s.m == s.m ? logz - s.b / (1.f + s.z) : NAN;
            if (a.tokens) a.logprob[row] = listed ? log_of(given) : 0.f;
        }
        if (TOP && lane < a.k) {
            a.top_ids[(size_t)row * a.k + lane] = (int32_t)~t.i;
            a.top_logprobs[(size_t)row * a.k + lane] = log_of(value(t.v));
        }
    };
    if (ADDERS == 1 ? warp == kWarps : warp >= kWarps && (warp == kWarps || a.rows - blockIdx.x > gridDim.x)) {
        turn = warp - kWarps;                  // row after row in turn
        for (uint32_t row = blockIdx.x / cluster + turn * gridDim.x;; turn += ADDERS) {
            const Run r = run_of(row);
            const uint32_t half = turn & 1;
            if (rank == 0) token_of(row);
            if (ok) ok = __all_sync(0xffffffffu, wait(there + 8 * half, (turn / 2) & 1));
            s = over_lanes(lane < kWarps ? part[half][lane] : Sums{-INFINITY, 0.f, 0.f});
            if constexpr (TOP) {
                // The k lanes (of the block) with the largest entries have the k largest entries among theirs, whatever is larger than the k-th lane's: in the
                // vector that holds the lane's largest, and where its others reach as high, in all of them.  (Order by value, then by vector: of equal
                // values in one vector all are taken.)  The lanes' largest are in order already; what is found beside them, not much as a rule, is put in.
                t = first_of(lists[half], a.k);
                const Top least = {__shfl_sync(0xffffffffu, t.v, a.k - 1), __shfl_sync(0xffffffffu, t.i, a.k - 1)};
                const uint4* const xv = reinterpret_cast<const uint4*>(r.x + r.head);
                const bool mine = lane < a.k && t.v;
                const uint32_t vec = ~t.i, of = mine ? (vec - r.v0) / kStageVecs % kWarps : 0, at = mine ? (vec - r.v0) % 32 : 0;
                Top found = {0, 0};
                auto offer = [&](float y, uint32_t vec, uint32_t id, bool in) {    // entry `id` of a lane's vector `vec`
                    const uint32_t o = order(y);
                    uint32_t who = __ballot_sync(0xffffffffu, in && (o > least.v || (o == least.v && ~vec >= least.i)));
                    while (who) {
                        const uint32_t from = __ffs(who) - 1;
                        who &= who - 1;
                        insert(found, __shfl_sync(0xffffffffu, o, from), __shfl_sync(0xffffffffu, ~id, from));
                    }
                };
                uint32_t first = 0xFFFFFFFFu;  // the lane's largest entry
                auto offer_vector = [&](const uint4& u, uint32_t vec, uint32_t but, bool in) {
                    float v[N];
                    Vec<T>::unpack(u, v);
#pragma unroll
                    for (uint32_t e = 0; e < N; e++) offer(v[e], vec, r.head + vec * N + e, in && r.head + vec * N + e != but);
                };
                const uint4 own = mine && ok ? xv[vec] : Vec<T>::nothing();
                if (mine && ok) {
                    float v[N];
                    Vec<T>::unpack(own, v);
#pragma unroll
                    for (uint32_t e = N; e > 0; e--)
                        if (order(v[e - 1]) == t.v) first = r.head + vec * N + e - 1;
                    found = Top{t.v, ~first};
                }
                const bool whole = mine && ok && seconds[half][of][at] >= least.v;
                offer_vector(own, vec, first, mine && ok && !whole);
                uint32_t again = __ballot_sync(0xffffffffu, whole);
                while (again) {
                    const uint32_t from = __ffs(again) - 1, f = r.v0 + __shfl_sync(0xffffffffu, of * kStageVecs + at, from), but = __shfl_sync(0xffffffffu, first, from);
                    again &= again - 1;
                    for (uint32_t j = lane; __any_sync(0xffffffffu, f + j / kAhead * kWarps * kStageVecs < r.v1); j += 32) {       // the lane's j-th vector
                        const uint32_t v = f + j / kAhead * kWarps * kStageVecs + j % kAhead * 32;
                        offer_vector(v < r.v1 ? xv[v] : Vec<T>::nothing(), v, but, v < r.v1);
                    }
                }
                // the entries outside of the vectors: those in front come before all others of their value, those behind after them
                if (rank == 0 && r.head) offer(lane < r.head ? to_f32(r.x[lane]) : 0.f, 0, lane, lane < r.head);
                if (rank == cluster - 1 && r.tail) {
                    const uint32_t id = r.head + r.vecs * N + lane;
                    offer(lane < r.tail ? to_f32(r.x[id]) : 0.f, r.vecs, id, lane < r.tail);
                }
                t = found;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(taken + 8 * half);
            if (cluster == 1) result(row);
            if (cluster > 1 || a.rows - row <= (uint64_t)ADDERS * gridDim.x) break;
            row += ADDERS * gridDim.x;
        }
        if (cluster > 1) {                     // to the first block
            if (lane == 0) {
                const uint32_t to = cluster_map(smem_u32(&blocks[rank]), 0);
                asm volatile("st.shared::cluster.f32 [%0], %1;\n st.shared::cluster.f32 [%0 + 4], %2;\n st.shared::cluster.f32 [%0 + 8], %3;" ::"r"(to), "f"(s.m), "f"(s.z), "f"(s.b) : "memory");
            }
            if (TOP) asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(cluster_map(smem_u32(&best[rank][lane]), 0)), "r"(t.v), "r"(t.i) : "memory");
        }
    }
    if (!ok && lane == 0 && a.status) atomicCAS(a.status, 0, 1);
    if (cluster > 1) {
        __syncwarp();
        cluster_sync();
        if (rank == 0 && warp == kWarps) {
            if (TOP) {                         // a block's list a lane
                uint32_t at = 0;
                Top x = lane < cluster ? best[lane][0] : Top{0, 0};
                t = largest(a.k, [&]() { return x; }, [&]() { x = ++at < 32 ? best[lane][at] : Top{0, 0}; });
            }
            s = over_lanes(lane < cluster ? blocks[lane] : Sums{-INFINITY, 0.f, 0.f});
            result(blockIdx.x / cluster);
        }
    }
}

// Blocks of a row: enough rows fill the GPU by themselves; a block has 2048 entries at least.
static uint32_t cluster_of(uint32_t rows, uint32_t n) {
    uint32_t c = 1;
    while (c < 16 && (uint64_t)rows * c * 2 <= 2 * 148 && n / (c * 2) >= 2048) c *= 2;
    return c;
}
template <typename T, bool TOP, uint32_t ADDERS> static int32_t launch(runit_ctx* ctx, const Args& a) {
    constexpr uint32_t smem = kWarps * kStages * kStageBytes;
    const uint32_t cluster = cluster_of(a.rows, a.n);
    static bool configured[64] = {false};
    if (ctx->device >= 64 || !configured[ctx->device]) {
        RUNIT_CUDA_TRY(ctx, cudaFuncSetAttribute(token_logprobs_kernel<T, TOP, ADDERS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        RUNIT_CUDA_TRY(ctx, cudaFuncSetAttribute(token_logprobs_kernel<T, TOP, ADDERS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        if (ctx->device < 64) configured[ctx->device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster > 1 ? a.rows * cluster : min(a.rows, (uint32_t)ctx->sm_count * kBlocksPerSm));
    cfg.dynamicSmemBytes = smem;
    cfg.blockDim = dim3(32 * (kWarps + ADDERS));
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->tune.pdl != 0 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, TOP, ADDERS>, a, cluster);           // errors surface in runit_after_launch
    return runit_after_launch(ctx, "token_logprobs");
}
// A second warp to add up where blocks have rows one behind the other and short ones, so that the alternatives take as long as the reading (4000 rows of 2000, 20
// alternatives: 64 us with one, 45 with two; 2048 rows of 152064 with 5: 119 and 122, both on one GPU).
template <typename T, bool TOP> static int32_t run(runit_ctx* ctx, const Args& a) {
    if constexpr (TOP)
        if (a.rows > (uint32_t)ctx->sm_count * kBlocksPerSm && a.n < 32768) return launch<T, TOP, 2>(ctx, a);
    return launch<T, TOP, 1>(ctx, a);
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
    const lp::Args a{logits, (const int32_t*)tokens, (float*)logprob, (float*)entropy, (float*)top_logprobs, (int32_t*)top_ids, ctx->d_status, ld, n, k, rows};
    if (type == RUNIT_TYPE_F32) return k ? lp::run<float, true>(ctx, a) : lp::run<float, false>(ctx, a);
    if (type == RUNIT_TYPE_F16) return k ? lp::run<__half, true>(ctx, a) : lp::run<__half, false>(ctx, a);
    return k ? lp::run<__nv_bfloat16, true>(ctx, a) : lp::run<__nv_bfloat16, false>(ctx, a);
}
