// What the kernels of the attention over a paged cache share: arguments, places in the scratch, the products of the legacy tensor path, and the
// operations on scores.
#pragma once

#include "gemv_common.cuh"
#include "paged.cuh"
#include "tma.cuh"

namespace runit {
namespace pg {

constexpr float kLog2e = 1.4426950408889634f;

struct Tanh {                // tanh_of
    float k, far, n[3], f[4];                  // far: the square of v from which on neither polynomial serves
};
struct AttnArgs {
    Cache c;
    const void* q;
    void* out;
    const float* slopes;
    uint32_t ldq, ldo, window;
    float scale, cap;
    Tanh tanh;               // of scale / cap times a product
    // scratch
    uint32_t* plan;          // kPlanHead words, then the steps in front of every entry
    float *slot_o, *slot_ml; // [2 * workers][16][dim] and [..][16][2]: pieces of segments that workers share
    float *row_o, *row_ml;   // [rows * heads][dim] and [..][2]: what one worker has of a row whose shared positions come from elsewhere
    float *pre_o, *pre_ml;   // the same for the shared positions
};
// What a launch of the kernel for many rows does (paged_attention_tc.cu): the shared positions for all rows, or every sequence's own positions.
struct TcArgs {
    uint32_t box, split;     // positions of a copy; parts that a tile's positions are cut into
    bool shared, direct;     // direct: a row is done with this launch
    bool beside;             // the launch in front belongs to the same call and has waited for what came before: nothing of it is read here
    float *part_o, *part_ml; // [split][rows * heads][dim] and [..][2]
};
int32_t paged_attention_tc(runit_ctx* ctx, const runit_paged_cfg* g, const AttnArgs& a, TcArgs w, uint32_t tiles);

__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int32_t c0, int32_t c1, int32_t c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory"); }
// What differs between the two 16-bit types: products, packing, bits that are no number, and their range.  Weights are 2^(s - ref) when they are rounded to the
// type, ref kLift below a row's largest score; in the kernel for many rows kLift - kRise below the one that was the largest when ref was set last, which scores may
// exceed by kRise.  f16 has ten bits down to 2^-14 only and nothing below 2^-25: with the largest weights at 2^15, those down to 2^-29 of the largest (2^-25 in the
// other kernel) are off by half a step relative to themselves, and 131072 weights below that, 2^-8 of the sum at most, by 2^-19 of it together.  (With the largest
// at 1, a row whose best key is 17 nats ahead of thousands of others lost up to all that the others have.)  bf16 has its eight bits throughout, and values up to the
// end of f32's range: no weight exceeds 1.
template <typename T> struct Half2;
template <> struct Half2<__half> {
    static constexpr float kLift = 15.f, kRise = 4.f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7FFF7FFFu) + 0x04000400u) & 0x80008000u; }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Half2<__nv_bfloat16> {
    static constexpr float kLift = 0.f, kRise = 8.f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
    static __device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7FFF7FFFu) + 0x00800080u) & 0x80008000u; }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
// the 16-bit halves of w that are no numbers, set to zero
template <typename T> __device__ __forceinline__ uint32_t finite_part(uint32_t w, uint32_t nf) { return w & ~((nf >> 15) * 0xFFFFu); }

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// tanh(k v) of N products.  tanh u = u p(u^2), p fitted to the least relative error (weighted least squares): of degree 2 below 0.25 (4.2e-7) and of degree 3
// below 0.5 (5.5e-7); the powers of k are in the coefficients.  Larger arguments take (1 - e^-2|u|) / (1 + e^-2|u|), off by some 2^-22; so does their whole warp,
// with u itself for those below 0.5, and every warp if powers of k leave the range.
static inline Tanh tanh_of(float k_) {
    const double k = k_, k2 = k * k;
    const bool in = k2 > 0x1p-34 && k2 < 0x1p34;
    Tanh h;
    h.k = k_;
    h.far = in ? (float)(0.25 / k2) : -1.f;
    h.n[0] = (float)(0.9999996 * k); h.n[1] = (float)(-0.33321908 * k * k2); h.n[2] = (float)(0.12841612 * k * k2 * k2);
    h.f[0] = (float)(0.99999946 * k); h.f[1] = (float)(-0.33326318 * k * k2); h.f[2] = (float)(0.13190296 * k * k2 * k2); h.f[3] = (float)(-0.04440222 * k * k2 * k2 * k2);
    return h;
}
// For a whole warp, which looks first how large the arguments are.
template <int N> __device__ __forceinline__ void tanh_scores(float (&v)[N], const Tanh& h) {
    uint64_t x[N / 2], w[N / 2];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        x[i] = pack2(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]));
        w[i] = fmul2(x[i], x[i]);
        most = max3(most, __uint_as_float((uint32_t)w[i]), __uint_as_float((uint32_t)(w[i] >> 32)));
    }
    if (!__any_sync(0xffffffffu, most > h.far)) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint64_t p = fmul2(x[i], ffma2(w[i], ffma2(w[i], ffma2(w[i], packf(h.f[3]), packf(h.f[2])), packf(h.f[1])), packf(h.f[0])));
            v[2 * i] = __uint_as_float((uint32_t)p);
            v[2 * i + 1] = __uint_as_float((uint32_t)(p >> 32));
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float u = v[i] * h.k, u2 = u * u, e = exp2_approx(-2.f * kLog2e * fabsf(u));
            const float small = u * fmaf(u2, fmaf(u2, fmaf(u2, -0.04440222f, 0.13190296f), -0.33326318f), 0.99999946f);
            v[i] = u2 < 0.25f ? small : copysignf(__fdividef(1.f - e, 1.f + e), u);
        }
    }
}
// Below 0.25; beyond it the result exceeds kNearTanh, as u p(u^2) rises throughout (its derivative 1 - u^2 + 0.64 u^4 has no zero).  four: the largest magnitudes.
constexpr float kNearTanh = 0.2449f;
template <int N> __device__ __forceinline__ void tanh_near(float (&v)[N], const Tanh& h, float (&four)[4]) {
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        const uint64_t x = pack2(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1])), w = fmul2(x, x);
        const uint64_t p = fmul2(x, ffma2(w, ffma2(w, packf(h.n[2]), packf(h.n[1])), packf(h.n[0])));
        v[2 * i] = __uint_as_float((uint32_t)p);
        v[2 * i + 1] = __uint_as_float((uint32_t)(p >> 32));
        four[i & 3] = max3(four[i & 3], fabsf(v[2 * i]), fabsf(v[2 * i + 1]));
    }
}
// The first position that the one at `pos` sees.
__device__ __forceinline__ uint32_t first_seen(int32_t pos, uint32_t window) { return window && pos >= 0 && (uint32_t)pos >= window ? (uint32_t)pos + 1 - window : 0; }
// Sequence of a row by halving the starts; c.n_seqs: nobody's.
__device__ __forceinline__ uint32_t sequence_by_halves(const Cache& c, uint32_t row) {
    uint32_t lo = 0, hi = c.n_seqs;            // as many of q_start[1 ..] as are <= row
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (c.q_start[mid + 1] <= (int32_t)row) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

}  // namespace pg
}  // namespace runit
