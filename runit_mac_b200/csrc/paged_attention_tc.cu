// Attention over a paged cache for many rows that share keys (prompts, and a prefix that a whole batch shares), on the tcgen05 tensor cores.
//
// A CTA has up to 256 (row, query head) pairs of one key head, as two tiles of 128, and walks a part of their positions in blocks of 128 that both tiles
// share.  By halves of a block, 64 positions, a tile has S = Q K^T in tensor memory (f32); four warps, a thread a row, read S (and free it for the next half),
// take its maximum, form the weights 2^(s - ref) and put them down as 16-bit numbers in one of two places; O += P V, accumulated in tensor memory, P
// being the A operand from there and V (as it lies in the cache) MN-major.  While the weights of one half are formed, the scores of the next one and the
// product of the last one run.  ref is a row's largest score until one exceeds it by 2^kRise, so that O is rarely scaled; the weights keep the
// relative error of their rounding (Half2), and sums of them are f32.
// Tensor memory, 512 columns: S 64 and P 2 x 32 of each tile, O 128 of each.
// Bound: products of 64 positions, whose operands from shared memory take 48 clocks instead of 32 (1260 a half for both tiles), and the warps of the softmax, which
// have 512 clocks of exponentials a half and some 1200 with all the rest, two of them a scheduler.  3584 (row, head) pairs over 32768 positions, dim 128:
// 71 us, 850 TFLOP/s; prompts of 3 x 700 .. 2048 rows behind 2048 .. 4096 positions, 16 heads of 128, scores capped, 115 to 118 us, 540 to 526 TFLOP/s (256
// tiles leave 148 SMs idle for a fifth of that: 38 blocks on the busiest, 30.8 on average).  Whole blocks of 128 positions at a time: 5% slower.
// K and V of a block come by TMA as boxes of whole pages or of 128 positions; positions outside of what the CTA's rows see are zeros in V.
#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace runit {
namespace pg {

constexpr uint32_t kTcRows = 256, kKeys = 128, kSoftWarps = 8, kTcThreads = 32 * (kSoftWarps + 3);   // and a warp for each tile's products, one for copies

template <int HD> struct TcShape {
    static constexpr uint32_t kPanel = 128 * 128;  // 64 elements of 128 rows
    static constexpr uint32_t kTile = HD / 64 * kPanel;
    static constexpr uint32_t kSlots = HD == 128 ? 5 : 8;      // of K and V blocks in turn
    static constexpr uint32_t kSmem = (2 + kSlots) * kTile + 1024;
};

__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr, uint32_t panel) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
template <typename T> __host__ __device__ constexpr uint32_t idesc_of(uint32_t m, uint32_t n, uint32_t b_mn);
template <> __host__ __device__ constexpr uint32_t idesc_of<__half>(uint32_t m, uint32_t n, uint32_t b_mn) { return umma_idesc_f16(m, n, b_mn); }
template <> __host__ __device__ constexpr uint32_t idesc_of<__nv_bfloat16>(uint32_t m, uint32_t n, uint32_t b_mn) { return umma_idesc_f16(m, n, b_mn) | (1u << 7) | (1u << 10); }

// One row's attention over positions lo .. hi of a table, by a warp with plain arithmetic: for rows whose products met a value that is no number at a
// position that they do not see (0 x Inf).  A lane takes the score of one of 32 positions, then the warp their values one by one.  Returns maximum (log2 units)
// and sum; o: HD / 32 of the dimensions per lane.
template <typename T, int HD>
__device__ __noinline__ float2 plain_row(const AttnArgs& a, const int32_t* table, uint32_t token, uint32_t head, int32_t pos, uint32_t lo, uint32_t hi, float* out) {
    constexpr uint32_t E = HD / 32;
    const Cache& c = a.c;
    const uint32_t lane = threadIdx.x & 31;
    const uint4* const qp = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (size_t)token * a.ldq + (size_t)head * HD);
    float o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (uint32_t e = 0; e < E; e++) o[e] = 0.f;
    const float slope = a.slopes ? a.slopes[head] : 0.f;
    for (uint32_t j0 = lo; j0 < hi; j0 += 32) {
        const uint32_t j = j0 + lane, n = min(32u, hi - j0);
        bool ok;
        const size_t at = page_row(c, table, min(j, hi - 1), head / c.group, &ok);
        const uint4* const kp = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(c.k) + at);
        float t = 0.f;
#pragma unroll 4
        for (uint32_t d = 0; d < HD / 8; d++) {
            const uint4 x = qp[d], y = kp[d];
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const float2 u = Half2<T>::unpack(reinterpret_cast<const uint32_t*>(&x)[e]), v = Half2<T>::unpack(reinterpret_cast<const uint32_t*>(&y)[e]);
                t = fmaf(u.x, v.x, t);
                t = fmaf(u.y, v.y, t);
            }
        }
        t *= a.scale;
        if (a.cap != 0.f) t = a.cap * tanhf(t / a.cap);
        t = lane < n ? (t - slope * (float)(pos - (int32_t)j)) * kLog2e : -INFINITY;
        float top = fmaxf(m, t);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float old = top == -INFINITY ? 1.f : exp2_approx(m - top), p = exp2_approx(top == -INFINITY ? t : t - top);
        float sum = p;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        l = fmaf(l, old, sum);
#pragma unroll
        for (uint32_t e = 0; e < E; e++) o[e] *= old;
#pragma unroll 4
        for (uint32_t i = 0; i < n; i++) {
            const float w = __shfl_sync(0xffffffffu, p, i);
            const T* const vp = reinterpret_cast<const T*>(c.v) + __shfl_sync(0xffffffffu, at, i) + lane * E;
#pragma unroll
            for (uint32_t e = 0; e < E; e++) o[e] = fmaf(w, to_f32(vp[e]), o[e]);
        }
        m = top;
    }
#pragma unroll
    for (uint32_t e = 0; e < E; e++) out[e] = o[e];
    return make_float2(m, l);
}
// The first and the last of the positions lo .. hi of a table that have a value of key head h which is no number, by a warp; {0xFFFFFFFF, 0}: none has.
template <typename T, int HD>
__device__ __noinline__ uint2 not_finite_values(const Cache& c, const int32_t* table, uint32_t h, uint32_t lo, uint32_t hi) {
    constexpr uint32_t CH = HD / 8;                // 16-byte pieces of a row
    const uint32_t lane = threadIdx.x & 31;
    uint32_t first = 0xFFFFFFFFu, last = 0;
#pragma unroll 4
    for (uint32_t j = lo + lane / CH; j < hi; j += 32 / CH) {
        bool ok;
        const uint4 x = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(c.v) + page_row(c, table, j, h, &ok))[lane % CH];
        if (Half2<T>::not_finite(x.x) | Half2<T>::not_finite(x.y) | Half2<T>::not_finite(x.z) | Half2<T>::not_finite(x.w)) {
            first = min(first, j);
            last = j;
        }
    }
    __syncwarp();
    return make_uint2(__reduce_min_sync(0xffffffffu, first), __reduce_max_sync(0xffffffffu, last));
}

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) attention_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const AttnArgs a, const TcArgs w) {
    using S = TcShape<HD>;
    constexpr float kRise = Half2<T>::kRise, kBelow = Half2<T>::kLift - kRise;       // weights are relative to ref - kBelow
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * S::kSlots + 14];
    __shared__ uint32_t tmem_holder, found[4], sums[kTcThreads / 32];
    __shared__ volatile int abort_flag;
    const Cache& c = a.c;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    // full, empty: one phase per use of a slot; p_full of a tile's halves: one per block; s_full, s_free, o_full, turn: one per half block; done: one
    const uint32_t full = smem_u32(bars), empty = full + 8 * S::kSlots, s_full = empty + 8 * S::kSlots, s_free = s_full + 16, p_full = s_free + 16, o_full = p_full + 32, done = o_full + 16, turn = done + 16;
    if (tid == 0) {
        prefetch_map(&mk);
        prefetch_map(&mv);
        abort_flag = 0;
        found[0] = 0xFFFFFFFFu;
        found[2] = c.shared;
        found[3] = 0;
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(&tmem_holder), 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_holder;
    if (w.beside) {
        acquire_ahead(c);
        asm volatile("fence.proxy.async.global;" ::: "memory");  // for the pages, which the copies read
    } else grid_dependency_wait();
    grid_launch_dependents();

    // which rows and positions
    const uint32_t part = blockIdx.x % w.split, h = blockIdx.x / w.split % c.kv_heads, index = blockIdx.x / w.split / c.kv_heads;
    if (w.shared) {
        uint32_t lo = c.shared, hi = 0;
        for (uint32_t e = tid; e < c.n_seqs; e += kTcThreads) {
            const Seq s = sequence(c, e);
            if (!s.n) continue;
            lo = min(lo, first_seen((int32_t)s.len - (int32_t)s.n, a.window));
            hi = max(hi, min(s.len, c.shared));
        }
        atomicMin(&found[2], lo);
        atomicMax(&found[3], hi);
        if (tid == 0) {
            found[0] = c.n_seqs;
            found[1] = index;
        }
    } else if (c.n_seqs <= 32) {               // all sequences' last tiles first, then those in front of them: those with the most positions begin
        if (warp == 0) {
            const uint32_t n = lane < c.n_seqs ? (sequence(c, lane).n * c.group + kTcRows - 1) / kTcRows : 0;
            if (index < __reduce_add_sync(0xffffffffu, n)) {
                uint32_t r = 0;                // tiles of every sequence that come before the one that is looked for
                for (uint32_t step = 1u << (31 - __clz(__reduce_max_sync(0xffffffffu, n))); step > 0; step /= 2)
                    if (__reduce_add_sync(0xffffffffu, min(n, r + step)) <= index) r += step;
                const uint32_t rest = index - __reduce_add_sync(0xffffffffu, min(n, r)), has = __ballot_sync(0xffffffffu, n > r);
                uint32_t e = has;
                for (uint32_t i = 0; i < rest; i++) e &= e - 1;
                e = __ffs(e) - 1;
                const uint32_t tiles = __shfl_sync(0xffffffffu, n, e);
                if (lane == 0) {
                    found[0] = e;
                    found[1] = tiles - 1 - r;
                }
            }
        }
    } else {                                   // tiles in front of a sequence; the last ones begin
        const uint32_t per = (c.n_seqs + kTcThreads - 1) / kTcThreads, beg = min(c.n_seqs, tid * per), end = min(c.n_seqs, beg + per);
        uint32_t sum = 0;
        for (uint32_t e = beg; e < end; e++) sum += (sequence(c, e).n * c.group + kTcRows - 1) / kTcRows;
        uint32_t inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += v;
        }
        if (lane == 31) sums[warp] = inc;
        __syncthreads();
        uint32_t off = inc - sum, total = 0;
        for (uint32_t i = 0; i < kTcThreads / 32; i++) {
            if (i < warp) off += sums[i];
            total += sums[i];
        }
        const uint32_t want = total - 1 - index;                 // beyond every tile where index >= total
        if (index < total && want >= off && want < off + sum) {
            uint32_t e = beg, at = off;
            for (;; e++) {
                const uint32_t n = (sequence(c, e).n * c.group + kTcRows - 1) / kTcRows;
                if (want < at + n) break;
                at += n;
            }
            found[0] = e;
            found[1] = want - at;
        }
    }
    // the starts of the sequences, where the copies go later: the shared positions' rows look for their sequences
    int32_t* const starts = reinterpret_cast<int32_t*>(smem_raw + (base - smem_u32(smem_raw)));
    if (w.shared)
        for (uint32_t e = tid; e <= c.n_seqs; e += kTcThreads) starts[e] = c.q_start[e];
    __syncthreads();
    const uint32_t entry = found[0], tile = found[1];
    uint32_t row0 = 0, n_pairs = c.rows * c.group, lo = 0, hi = 0;
    int32_t base_pos = 0;
    const int32_t* table = c.table;
    if (w.shared) {
        lo = found[2];
        hi = found[3];
    } else if (entry != 0xFFFFFFFFu) {
        const Seq s = sequence(c, entry);
        row0 = s.row0;
        n_pairs = s.n * c.group;
        base_pos = (int32_t)s.len - (int32_t)s.n;
        const uint32_t last = min(n_pairs, (tile + 1) * kTcRows) - 1;
        lo = max(c.shared, first_seen(base_pos + (int32_t)(tile * kTcRows / c.group), a.window));
        hi = (uint32_t)max(0, base_pos + (int32_t)(last / c.group) + 1);
        table += (size_t)entry * c.table_ld;
        if (tid == 0) {                        // for whoever looks for values that are no numbers, in the end
            found[2] = lo;
            found[3] = hi;
        }
    }
    const bool any = entry != 0xFFFFFFFFu && tile * kTcRows < n_pairs;
    const uint32_t first_row = tile * kTcRows, start = lo & ~(w.box - 1), steps = any && hi > lo ? (hi - start + kKeys - 1) / kKeys : 0;
    const uint32_t b0 = (uint32_t)((uint64_t)part * steps / w.split), n_blocks = (uint32_t)((uint64_t)(part + 1) * steps / w.split) - b0;
    const uint32_t chains = any && n_pairs - first_row > 128 ? 2 : 1;
    bool ok = true;
    // the row of a softmax thread
    const uint32_t chain = warp >> 2, row = tid & 127, pair = first_row + chain * 128 + row;
    bool live = warp < kSoftWarps && any && pair < n_pairs;
    const uint32_t token = row0 + (live ? pair / c.group : 0), head = h * c.group + (live ? pair % c.group : 0);
    int32_t pos = base_pos + (int32_t)(pair / c.group);
    if (w.shared && live) {
        uint32_t s = 0;
        for (uint32_t n = 4096; n > 0; n /= 2)           // as many of starts[1 ..] as are <= token
            if (s + n <= c.n_seqs && starts[s + n] <= (int32_t)token) s += n;
        live = s < c.n_seqs;
        if (live) {
            const Seq q = sequence(c, s);
            live = token >= q.row0 && token < q.row0 + q.n;
            pos = (int32_t)q.len - (int32_t)(q.row0 + q.n - token);
        }
    }
    // a barrier a lane
    if (warp == kSoftWarps + 2) {
        constexpr uint32_t n = 2 * S::kSlots;
        const uint32_t i = lane - n;           // behind full and empty: s_full, s_free, p_full, o_full, done, turn
        if (lane < n + 14) mbar_init(full + 8 * lane, lane < S::kSlots ? 1 : lane < n ? chains : i < 2 ? 1 : i < 4 ? 4 : i < 8 ? 128 : i < 12 ? 1 : 4);
        fence_mbar_init();
    }
    // Q, asked for before anything is waited for
    constexpr uint32_t CH = HD / 8, RW = 32 / CH;                // 16-byte pieces of a row; rows that a warp reads at once
    const uint32_t ch = lane % CH;
    uint4 q_in[32 / RW];
    if (warp < kSoftWarps) {
#pragma unroll
        for (uint32_t i = 0; i < 32 / RW; i++) {
            const uint32_t r = i * RW + lane / CH, tk = __shfl_sync(0xffffffffu, token, r), hd = __shfl_sync(0xffffffffu, head, r);
            const bool there = __shfl_sync(0xffffffffu, (int)live, r) != 0;
            q_in[i] = there ? reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (size_t)tk * a.ldq + (size_t)hd * HD)[ch] : make_uint4(0, 0, 0, 0);
        }
    }
    __syncthreads();

    if (warp == kSoftWarps + 2) {              // copies: K(0), V(0), K(1), ... into the slots in turn
        uint32_t n = 0;
        const uint32_t boxes = kKeys / w.box;
        for (uint32_t j = 0; j < n_blocks && ok; j++) {
            const uint32_t k0 = start + (b0 + j) * kKeys, k = k0 + lane * w.box;
            const bool mine = lane < boxes && k < hi && k + w.box > lo;
            int32_t page = mine ? table[k >> c.page_log2] : 0;
            if ((uint32_t)page >= c.n_pages) {
                report(c);
                page = 0;
            }
            const int32_t row = (int32_t)((((uint32_t)page * c.kv_heads + h) << c.page_log2) + (k & ((1u << c.page_log2) - 1)));
            const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine)) * w.box * HD * 2;
            for (uint32_t v = 0; v < 2 && ok; v++, n++) {
                const uint32_t slot = n % S::kSlots, bar = full + 8 * slot, dst = base + (2 + slot) * S::kTile;
                if (n >= S::kSlots) ok = mbar_wait_timed(empty + 8 * slot, (n / S::kSlots - 1) & 1, &abort_flag);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                if (lane == 0) mbar_expect_tx(bar, bytes);
                __syncwarp();
                if (mine)
                    for (uint32_t p = 0; p < HD / 64; p++) tma_load_2d(dst + p * S::kPanel + lane * w.box * 128, v ? &mv : &mk, 128 * p, row, bar);
                __syncwarp();
            }
        }
        // nothing is in flight when the block leaves
        mbar_drain(full, S::kSlots, n);
    } else if (warp >= kSoftWarps) {           // a tile's products
        const uint32_t i = warp - kSoftWarps, qs = base + i * S::kTile, s_cols = tmem + 64 * i, p_cols = tmem + 128 + 64 * i, o_cols = tmem + 256 + 128 * i;
        const uint32_t halves = i < chains ? 2 * n_blocks : 0;
        uint32_t n_s = 0, n_o = 0, n_d = 0;
        auto slot_of_use = [&](uint32_t n) { return base + (2 + n % S::kSlots) * S::kTile; };
        auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = ok && mbar_wait_timed(bar, parity, &abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after_sync();
        };
        auto wait_full = [&](uint32_t n) { wait(full + 8 * (n % S::kSlots), (n / S::kSlots) & 1); };
        // half h of a block's scores, with the block of K that is use n; the slot is free behind the second one
        auto scores = [&](uint32_t n, uint32_t h) {
            const uint32_t kb = slot_of_use(n) + 8192 * h;
            if (elect_one()) {
#pragma unroll
                for (int s = 0; s < HD / 16; s++) {
                    const uint32_t off = (s >> 2) * S::kPanel + (s & 3) * 32;
                    umma_bf16(s_cols, umma_desc_sw128(qs + off), umma_desc_sw128(kb + off), idesc_of<T>(128, kKeys / 2, 0), s > 0);
                }
                umma_commit(s_full + 8 * i);
                if (h) umma_commit(empty + 8 * (n % S::kSlots));
            }
            __syncwarp();
            n_s++;
        };
        asm volatile("bar.sync 1, 320;" ::: "memory");           // Q is there
        tc_fence_after_sync();
        if (halves) {
            wait_full(0);
            if (ok) scores(0, 0);
        }
        for (uint32_t n = 0; n < halves && ok; n++) {
            const uint32_t j = n >> 1, h = n & 1, uv = 2 * j + 1, uk = 2 * j + 2, k0 = start + (b0 + j) * kKeys, vb = slot_of_use(uv);
            const bool last = n + 1 == halves;
            if (!last) {                       // the next half's scores, as soon as this one's have been read
                if (h) wait_full(uk);
                wait(s_free + 8 * i, n & 1);
                if (!ok) break;
                scores(h ? uk : uk - 2, h ^ 1);
            }
            if (h == 0) {
                wait_full(uv);
                if (!ok) break;
                if (k0 < lo || k0 + kKeys > hi) {                // zeros where no row looks: the copies have left there what lay there, or the neighbours of what was asked for
                    const uint32_t from = lo > k0 ? lo - k0 : 0, to = hi - k0;
                    for (uint32_t x = lane; x < kKeys * (HD / 8); x += 32) {
                        const uint32_t r = x / (HD / 8), ch = x % (HD / 8);
                        if (r >= from && r < to) continue;
                        *reinterpret_cast<uint4*>(smem_raw + (vb - smem_u32(smem_raw)) + (ch >> 3) * S::kPanel + r * 128 + ((ch & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                    __syncwarp();
                }
            }
            wait(p_full + 16 * i + 8 * h, j & 1);
            if (!ok) break;
            if (elect_one()) {
#pragma unroll
                for (int s = 0; s < 4; s++)
                    umma_f16_ts(o_cols, p_cols + 32 * h + 8 * s, desc_mn_sw128(vb + (4 * h + s) * 2048, S::kPanel), idesc_of<T>(128, HD, 1), n > 0 || s > 0);
                umma_commit(last ? done + 8 * i : o_full + 8 * i);
                if (h && !last) umma_commit(empty + 8 * (uv % S::kSlots));
            }
            __syncwarp();
            if (last) {
                n_d++;
                break;
            }
            n_o++;
        }
        mbar_drain(s_full + 8 * i, 1, n_s);                      // nor is a product when the tensor memory goes back
        mbar_drain(o_full + 8 * i, 1, n_o);
        mbar_drain(done + 8 * i, 1, n_d);
    } else {
        const uint32_t lanes = (warp & 3) << 21, s_cols = tmem + 64 * chain + lanes, p_cols = tmem + 128 + 64 * chain + lanes, o_cols = tmem + 256 + 128 * chain + lanes;
        const uint32_t limit = w.shared ? c.shared : 0x7FFFFFFFu;
        const uint32_t row_lo = !live ? 0 : max(w.shared ? 0 : c.shared, first_seen(pos, a.window)), row_hi = !live ? 0x7FFFFFFFu : min((uint32_t)max(0, pos + 1), limit);
        const float slope = a.slopes && live ? a.slopes[head] : 0.f;
        {
            uint8_t* const dst = smem_raw + (base - smem_u32(smem_raw)) + chain * S::kTile + (warp & 3) * 32 * 128;
#pragma unroll
            for (uint32_t i = 0; i < 32 / RW; i++) {
                const uint32_t r = i * RW + lane / CH;
                *reinterpret_cast<uint4*>(dst + (ch >> 3) * S::kPanel + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = q_in[i];
            }
            fence_proxy_async();
        }
        asm volatile("bar.sync 1, 320;" ::: "memory");
        // plain: what the products (or their tanh) are multiplied by is positive, and nothing is added
        const float pre = a.cap != 0.f ? a.cap : a.scale;
        const bool plain = !a.slopes && pre > 0.f;
        const float mul = plain ? pre * kLog2e : kLog2e;
        float ref = -INFINITY, l = 0.f;
        bool wide = a.tanh.far < 0.f;          // some score is beyond the near polynomial
        bool cut = false;                      // some block had positions that this row does not see
        if (chain < chains) {
            for (uint32_t n = 0; n < 2 * n_blocks; n++) {
                const uint32_t h = n & 1, k0 = start + (b0 + (n >> 1)) * kKeys + 64 * h;
                if (ok) ok = mbar_wait_timed(s_full + 8 * chain, n & 1, &abort_flag);
                __syncwarp();
                tc_fence_after_sync();
                const bool inside = k0 >= row_lo && k0 + 64 <= row_hi;
                cut |= !inside;
                uint32_t r[2][32];
                tmem_ld32(s_cols, r[0]);
                tmem_ld32(s_cols + 32, r[1]);
                tmem_ld_wait();
                if (a.cap != 0.f) {
                    // The near polynomial grows with its argument, so that what comes out tells whether it was near: no vote ahead of it (7% of the time of the prompts
                    // above).  Scores that were not are read again, and a warp that has met one looks first from then on.
                    if (!wide) {
                        float four[4] = {0.f, 0.f, 0.f, 0.f};
                        tanh_near(reinterpret_cast<float(&)[32]>(r[0]), a.tanh, four);
                        tanh_near(reinterpret_cast<float(&)[32]>(r[1]), a.tanh, four);
                        wide = __any_sync(0xffffffffu, max3(fmaxf(four[0], four[1]), four[2], four[3]) > kNearTanh);
                        if (wide) {
                            tmem_ld32(s_cols, r[0]);
                            tmem_ld32(s_cols + 32, r[1]);
                            tmem_ld_wait();
                        }
                    }
                    if (wide) {
                        tanh_scores(reinterpret_cast<float(&)[32]>(r[0]), a.tanh);
                        tanh_scores(reinterpret_cast<float(&)[32]>(r[1]), a.tanh);
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free + 8 * chain);
                // scores, of which `mul` times are in units of log2
                if (!__all_sync(0xffffffffu, plain && inside)) {
#pragma unroll
                    for (uint32_t q = 0; q < 2; q++) {
                        if (!plain) {
                            const float at_0 = -slope * (float)(pos - (int32_t)(k0 + 32 * q));
#pragma unroll
                            for (int e = 0; e < 32; e++) r[q][e] = __float_as_uint(fmaf(__uint_as_float(r[q][e]), pre, fmaf(slope, (float)e, at_0)));
                        }
                    }
                    if (!__all_sync(0xffffffffu, inside)) {
#pragma unroll
                        for (uint32_t q = 0; q < 2; q++)
#pragma unroll
                            for (int e = 0; e < 32; e++) {
                                const uint32_t key = k0 + 32 * q + e;
                                if (key < row_lo || key >= row_hi) r[q][e] = 0xFF800000u;
                            }
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int q = 0; q < 2; q++)
#pragma unroll
                    for (int e = 0; e < 32; e += 2) mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], __uint_as_float(r[q][e]), __uint_as_float(r[q][e + 1]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mul;
                const bool rise = top > ref + kRise || (ref == -INFINITY && top > ref);
                const bool some = __any_sync(0xffffffffu, rise);
                float corr = 1.f;
                if (some) {
                    corr = rise ? exp2_approx(ref - top) : 1.f;
                    l *= corr;
                    ref = rise ? top : ref;
                }
                if (some && n > 0) {
                    // O with the last half's product: the one before it is behind these scores, so one of two phases is on
                    if (ok) ok = mbar_wait_timed(o_full + 8 * chain, (n - 1) & 1, &abort_flag);
                    __syncwarp();
                    tc_fence_after_sync();
#pragma unroll 1
                    for (int q = 0; q < HD / 16; q++) {
                        uint32_t o[16];
                        tmem_ld16(o_cols + 16 * q, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        tmem_st16(o_cols + 16 * q, o);
                    }
                }
                const float sub = ref == -INFINITY ? 0.f : ref - kBelow;
                const uint64_t mul2 = packf(mul), sub2 = packf(-sub);
                uint64_t both = 0;
                // The tiles take their exponentials in turn (half n of the second one once half n of the first is half done, and that behind half n - 1 of the
                // second).  Left alone they fall into step and do everything side by side (3 to 7% slower).
                if (ok && chains == 2 && (chain == 1 || n > 0)) ok = mbar_wait_timed(turn + 8 * chain, (chain == 1 ? n : n - 1) & 1, &abort_flag);
                __syncwarp();
                // The weights meet the values in the cache's type: half a step of it, relative, each (Half2: how far down); their sum is that of the 32-bit ones.
#pragma unroll
                for (uint32_t q = 0; q < 2; q++) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const uint64_t x = ffma2(pack2(r[q][2 * e], r[q][2 * e + 1]), mul2, sub2);
                        const float p0 = exp2_approx(__uint_as_float((uint32_t)x)), p1 = exp2_approx(__uint_as_float((uint32_t)(x >> 32)));
                        both = fadd2(both, pack2(__float_as_uint(p0), __float_as_uint(p1)));
                        p[e] = Half2<T>::pack(p0, p1);
                    }
                    tmem_st16(p_cols + 32 * h + 16 * q, p);
                    if (q == 0 && lane == 0) mbar_arrive(turn + 8 * (chain ^ 1));
                }
                tmem_st_wait();
                tc_fence_before_sync();
                mbar_arrive(p_full + 16 * chain + 8 * h);
                l += sum2(both);
            }
            if (n_blocks > 0 && ok) ok = mbar_wait_timed(done + 8 * chain, 0, &abort_flag);
            __syncwarp();
            tc_fence_after_sync();
            // The row's result: final, or this part's sums.  By way of shared memory (the warp's rows of Q, which all products have read): pieces of 64 bytes of 8
            // rows at a time; a thread's own row, 16 bytes at a time, would be as many half-written sectors (12000 clocks, now 5800).
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const size_t orow = (size_t)token * c.heads + head;
            float* const pml = w.part_ml + ((size_t)part * c.rows * c.heads + orow) * 2;
            uint8_t* const stage = smem_raw + (base - smem_u32(smem_raw)) + chain * S::kTile + (warp & 3) * (S::kTile / 4);
            const size_t to = w.direct ? (size_t)token * a.ldo * 2 + (size_t)head * HD * 2 : ((size_t)part * c.rows * c.heads + orow) * HD * 4;      // in bytes
            uint8_t* const out = w.direct ? reinterpret_cast<uint8_t*>(a.out) : reinterpret_cast<uint8_t*>(w.part_o);
            bool odd = false;
            auto pieces = [&](const uint32_t (&x)[16], uint32_t at) {        // 64 bytes of every row, `at` bytes from its begin
#pragma unroll
                for (int e = 0; e < 4; e++) *reinterpret_cast<uint4*>(stage + lane * 80 + 16 * e) = make_uint4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t r = 8 * e + lane / 4;
                    const size_t dst = __shfl_sync(0xffffffffu, to, r);
                    const bool there = __shfl_sync(0xffffffffu, (int)(live && ok), r) != 0;
                    if (there) *reinterpret_cast<uint4*>(out + dst + at + 16 * (lane % 4)) = *reinterpret_cast<const uint4*>(stage + r * 80 + 16 * (lane % 4));
                }
                __syncwarp();
            };
#pragma unroll 1
            for (int q = 0; q < HD / 32; q++) {
                uint32_t o[32];
                if (n_blocks > 0) {
                    tmem_ld32(o_cols + 32 * q, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0;
                }
#pragma unroll
                for (int e = 0; e < 32; e++) odd |= !(fabsf(__uint_as_float(o[e])) < INFINITY);
                uint32_t x[16];
                if (w.direct) {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = Half2<T>::pack(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
                    pieces(x, 64 * q);
                } else {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
#pragma unroll
                        for (int e = 0; e < 16; e++) x[e] = o[16 * i + e];
                        pieces(x, 128 * q + 64 * i);
                    }
                }
            }
            if (live && ok && !w.direct) *reinterpret_cast<float2*>(pml) = make_float2(ref - kBelow, l);
            // Rows with a result that is no number, and whether that is theirs: only if all such values lie where the row looks.  Looked for where one of these
            // rows does not look: beside the diagonal, as a rule, not the row's own positions, which are as many as the cache has.  (1024 rows over 3000 positions, 64
            // heads of 128, an infinite value in the middle that all rows see: 0.19 ms, 142 with all rows done again, 0.13 without it; at the last position, where
            // only one row sees it and the rest of its tile is done again: 29 ms.)
            uint32_t again = __ballot_sync(0xffffffffu, live && ok && odd && cut);
            if (again) {
                const bool mine = again >> lane & 1;
                const uint32_t from = max(found[2], start + b0 * kKeys), to = min(found[3], start + (b0 + n_blocks) * kKeys);
                const uint32_t front = min(to, __reduce_max_sync(0xffffffffu, mine ? row_lo : 0)), behind = max(from, __reduce_min_sync(0xffffffffu, mine ? row_hi : 0xFFFFFFFFu));
                const uint2 x = not_finite_values<T, HD>(c, table, h, from, front), y = not_finite_values<T, HD>(c, table, h, behind, to);
                again = __ballot_sync(0xffffffffu, mine && (x.x < row_lo || (y.x <= y.y && y.y >= row_hi)));
            }
            while (again) {
                const uint32_t from = __ffs(again) - 1;
                again &= again - 1;
                const uint32_t tk = __shfl_sync(0xffffffffu, token, from), hd = __shfl_sync(0xffffffffu, head, from);
                const uint32_t k_lo = max(__shfl_sync(0xffffffffu, row_lo, from), start + b0 * kKeys), k_hi = min(__shfl_sync(0xffffffffu, row_hi, from), start + (b0 + n_blocks) * kKeys);
                float x[HD / 32];
                const float2 ml = plain_row<T, HD>(a, table, tk, hd, __shfl_sync(0xffffffffu, pos, from), k_lo, k_hi, x);
                const size_t at = (size_t)tk * c.heads + hd;
                const float f = w.direct ? (ml.y == 0.f ? 0.f : 1.f / ml.y) : 1.f;
                for (uint32_t e = 0; e < HD / 32; e++) {
                    const uint32_t d = lane * (HD / 32) + e;
                    if (w.direct) (reinterpret_cast<T*>(a.out) + (size_t)tk * a.ldo + (size_t)hd * HD)[d] = from_f32<T>(x[e] * f);
                    else w.part_o[((size_t)part * c.rows * c.heads + at) * HD + d] = x[e];
                }
                if (!w.direct && lane == 0) *reinterpret_cast<float2*>(w.part_ml + ((size_t)part * c.rows * c.heads + at) * 2) = ml;
                __syncwarp();
            }
        }
    }
    if (!ok) {
        abort_flag = 1;
        if (c.status) atomicCAS(c.status, 0, 1);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
    if (w.beside) grid_dependency_wait();      // whoever waits for this launch waits for the one in front, too
}

template <typename T, int HD>
static int32_t run_tc(runit_ctx* ctx, const runit_paged_cfg* g, const AttnArgs& a, TcArgs w, uint32_t tiles) {
    static bool configured[64] = {false};
    if (ctx->device >= 64 || !configured[ctx->device]) {
        RUNIT_CUDA_TRY(ctx, cudaFuncSetAttribute(attention_tc_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<HD>::kSmem));
        if (ctx->device < 64) configured[ctx->device] = true;
    }
    CUtensorMap m[2];
    for (int i = 0; i < 2; i++) {
        const int32_t st = runit_get_tmap(ctx, i ? g->v_pages : g->k_pages, (uint64_t)g->n_pages * g->kv_heads * g->page, HD * 2, w.box, 128, &m[i], 1);
        if (st != RUNIT_OK) return st;
    }
    runit_launch_chain_smem(ctx, attention_tc_kernel<T, HD>, dim3(tiles * g->kv_heads * w.split), dim3(kTcThreads), TcShape<HD>::kSmem, m[0], m[1], a, w);
    return runit_after_launch(ctx, "paged_attention (many rows)");
}

int32_t paged_attention_tc(runit_ctx* ctx, const runit_paged_cfg* g, const AttnArgs& a, TcArgs w, uint32_t tiles) {
    if (g->type == RUNIT_TYPE_F16) return g->dim == 128 ? run_tc<__half, 128>(ctx, g, a, w, tiles) : run_tc<__half, 64>(ctx, g, a, w, tiles);
    return g->dim == 128 ? run_tc<__nv_bfloat16, 128>(ctx, g, a, w, tiles) : run_tc<__nv_bfloat16, 64>(ctx, g, a, w, tiles);
}

}  // namespace pg
}  // namespace runit
