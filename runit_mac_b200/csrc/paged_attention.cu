// Attention of a batch of sequences over a paged cache: out_i = sum_j softmax_j(s_ij) v_j over the positions j that row i sees, s_ij = scale q_i . k_j,
// then cap * tanh(s / cap), then minus slope * (i - j).
//
// Many rows that share keys: paged_attention_tc.cu.  Few rows a sequence (decoding): bound by HBM, which has to deliver every key and value once (one row over
// 131072 positions, 4 key heads of 128, f16: 268 MB in 51 us, 5.2 TB/s, of which 5 us are merge_kernel and 3 the way to the first copy; 64 sequences of
// 60 to 8100 positions, 206 MB: 44 us, 4.7 TB/s).  A segment is what shares keys: up to 16 (row, query head)
// pairs of one sequence and key head, and the positions that they see; the segments' steps of 32 positions, one behind the other, are dealt out evenly to
// the warps of the grid, whatever the lengths.  A warp is on its own: it copies its steps by TMA into a ring (boxes of 16 positions, so that pages of
// 16 are whole boxes), multiplies on the legacy tensor path with the rows as m16 (a tcgen05 tile would be 128 rows, mostly padding), and keeps
// maximum, sum and output of the running softmax in registers.  Segments that a warp has whole are done with that; the others leave a piece per warp, and
// merge_kernel adds them up.
#include "paged_attention.cuh"

namespace runit {
namespace pg {

constexpr uint32_t kWarps = 4, kStep = 32, kBox = 16, kRows = 16, kPlanHead = 16;
constexpr uint32_t kMaxWorkers = kWarps * 256;
constexpr uint32_t kStepsMin = 2;              // a worker's share at least: what it costs to begin and to merge is that of about two steps
constexpr uint32_t kFew = 256;                 // up to so many entries every warp finds its place for itself, without meeting the others
// Up to so many, merge_kernel works out the plan for itself while the split kernel runs; else it is left in the scratch (64 sequences 47.7 -> 46.5 us; 128
// behind shared positions, 3584 rows, 104.6 without and 105.3 with: too many warps, on SMs that are at work).
constexpr uint32_t kFewMerged = 64;

template <int HD> struct Shape {
    static constexpr uint32_t kBoxBytes = kBox * HD * 2, kStage = 4 * kBoxBytes, kStages = HD == 128 ? 3 : 6;
    static constexpr uint32_t kRing = kStage * kStages * kWarps;
};

// ── segments ──
// Entry e < n_seqs: a sequence and its own positions (from c.shared on); entry n_seqs (with shared positions): all rows and the shared ones.
struct Entry {
    uint32_t row0, n, tiles, lo, hi, steps;    // steps of one (key head, tile): the positions lo (down to a box) .. hi that any row of it sees
    int32_t base;                              // position of its first row
    const int32_t* table;
};
// Three more than its positions take, about what beginning and ending a segment costs a worker (64 sequences of 60 to 8100 positions: 113000 clocks for those
// with eight segments, 83000 for those with one; 77 us without, 64 with one step more, 60 with three).
__device__ __forceinline__ uint32_t steps_of(uint32_t lo, uint32_t hi) { return hi > lo ? (hi - (lo & ~(kBox - 1)) + kStep - 1) / kStep + 3 : 0; }
__device__ __forceinline__ Entry entry_of(const AttnArgs& a, uint32_t e, uint32_t pre_lo, uint32_t pre_hi, bool& falls) {
    const Cache& c = a.c;
    Entry t;
    if (e < c.n_seqs) {
        const Seq s = sequence(c, e);
        falls |= s.falls;
        t.row0 = s.row0;
        t.n = s.n;
        t.base = (int32_t)s.len - (int32_t)s.n;
        t.lo = max(c.shared, first_seen(t.base, a.window));
        t.hi = s.n ? s.len : 0;
        t.table = c.table + (size_t)e * c.table_ld;
    } else {
        t.row0 = 0;
        t.n = c.rows;
        t.base = 0;
        t.lo = pre_lo;
        t.hi = pre_hi;
        t.table = c.table;
    }
    t.tiles = (t.n * c.group + kRows - 1) / kRows;
    t.steps = steps_of(t.lo, t.hi);
    return t;
}
__device__ __forceinline__ Entry entry_of(const AttnArgs& a, uint32_t e, uint32_t pre_lo, uint32_t pre_hi) {
    bool falls = false;
    return entry_of(a, e, pre_lo, pre_hi, falls);
}
// Where starts fall (sequence() reports it), sequences overlap, and their steps can be too many for 32 bits: shares of a wrapped count would lie anywhere.  Whoever
// counts the steps learns of it here, and deals out nothing.
__device__ __forceinline__ uint32_t cost_of(const AttnArgs& a, uint32_t e, uint32_t pre_lo, uint32_t pre_hi, bool& falls) {
    const Entry t = entry_of(a, e, pre_lo, pre_hi, falls);
    return t.tiles * t.steps * a.c.kv_heads;
}
__device__ __forceinline__ uint32_t cost_of(const AttnArgs& a, uint32_t e, uint32_t pre_lo, uint32_t pre_hi) {
    bool falls = false;
    return cost_of(a, e, pre_lo, pre_hi, falls);
}
// The shared positions that some row of sequences e, e + step, ... sees.
__device__ __forceinline__ void seen_of(const AttnArgs& a, uint32_t e, uint32_t step, uint32_t& lo, uint32_t& hi) {
    for (; e < a.c.n_seqs; e += step) {
        const Seq s = sequence(a.c, e);
        if (!s.n) continue;
        lo = min(lo, first_seen((int32_t)s.len - (int32_t)s.n, a.window));
        hi = max(hi, min(s.len, a.c.shared));
    }
}
// Worker w of `workers` has the steps from begin_of(w) to begin_of(w + 1): the first ones have one more than the others.
__device__ __forceinline__ uint32_t begin_of(uint32_t w, uint32_t total, uint32_t workers) { return w * (total / workers) + min(w, total % workers); }
__device__ __forceinline__ uint32_t owner_of(uint32_t step, uint32_t total, uint32_t workers) {
    const uint32_t each = total / workers, more = total % workers, mid = more * (each + 1);
    return step < mid ? step / (each + 1) : more + (step - mid) / each;
}
__device__ __forceinline__ uint32_t workers_of(uint32_t total, uint32_t most) { return max(1u, min(most, total / kStepsMin)); }

struct Piece {
    float *o, *ml;
};
__device__ __forceinline__ Piece slot_of(const AttnArgs& a, uint32_t w, bool first) {
    const size_t s = 2 * (size_t)w + (first ? 0 : 1);
    return Piece{a.slot_o + s * kRows * a.c.dim, a.slot_ml + s * kRows * 2};
}

// V of a step whose hidden positions hold something that is no number: its elements were left out of the products (0 there), the rows that see
// them get them here.  p: the weights as the products' accumulators hold them.
template <typename T, int HD>
__device__ __noinline__ void add_not_finite(const uint8_t* stage_v, uint32_t k0, uint32_t end, const uint32_t (&lo)[2], const uint32_t (&hi)[2], const float (&p)[kStep / 8][4],
                                            float (&o)[HD / 8][4]) {
    const uint32_t lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll 1
    for (uint32_t j = 0; j < kStep; j++) {
        const uint32_t key = k0 + j;
        if (key >= end) break;                 // nothing behind that was copied
        float w[2] = {0.f, 0.f};
#pragma unroll
        for (uint32_t n = 0; n < kStep / 8; n++)
#pragma unroll
            for (uint32_t e = 0; e < 2; e++) {
                const float x = __shfl_sync(0xffffffffu, p[n][e], (lane & ~3u) | ((j & 7) >> 1)), y = __shfl_sync(0xffffffffu, p[n][2 + e], (lane & ~3u) | ((j & 7) >> 1));
                if (n == j / 8 && e == (j & 1)) { w[0] = x; w[1] = y; }
            }
        const uint32_t row = j % kBox;
        const uint8_t* box = stage_v + (j / kBox) * Shape<HD>::kBoxBytes;
#pragma unroll
        for (uint32_t d = 0; d < HD / 8; d++) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(box + (d >> 3) * (kBox * 128) + row * 128 + (((d & 7) ^ (row & 7)) << 4) + 4 * t);
            const uint32_t nf = Half2<T>::not_finite(word);
            if (!nf) continue;
            const float2 v = Half2<T>::unpack(word);
#pragma unroll
            for (uint32_t r = 0; r < 2; r++) {
                if (key < lo[r] || key >= hi[r]) continue;
                if (nf & 0x8000u) o[d][2 * r] += w[r] * v.x;
                if (nf & 0x80000000u) o[d][2 * r + 1] += w[r] * v.y;
            }
        }
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kWarps * 32, 1) paged_split_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const AttnArgs a,
                                                                   const uint32_t n_entries) {
    using S = Shape<HD>;
    constexpr uint32_t KS = HD / 16, ND = HD / 8, NK = kStep / 8;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[kWarps * S::kStages];
    __shared__ uint32_t sums[kWarps], edge[2], costs[kWarps][kFew];
    uint8_t* const ring = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
    uint32_t* const before = reinterpret_cast<uint32_t*>(ring + S::kRing);         // [n_entries + 1] steps in front of an entry
    const Cache& c = a.c;
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g4 = lane >> 2, t4 = lane & 3;
    if (tid == 0) {
        prefetch_map(&mk);
        prefetch_map(&mv);
    }
    if (tid < kWarps * S::kStages) mbar_init(smem_u32(&bars[tid]), 1);
    if (tid == 0) {
        edge[0] = c.shared;
        edge[1] = 0;
    }
    fence_mbar_init();
    __syncthreads();
    grid_dependency_wait();
    grid_launch_dependents();
    uint32_t pre_lo = c.shared, pre_hi = 0, total = 0, workers, me = warp * gridDim.x + blockIdx.x, x0, x1, e_first = 0, e_before = 0;
    // neighbours in the order of steps sit on other SMs: few steps spread over all of them
    auto share = [&]() {
        workers = workers_of(total, gridDim.x * kWarps);
        x0 = me < workers && total ? begin_of(me, total, workers) : 0;
        x1 = me < workers && total ? begin_of(me + 1, total, workers) : 0;
    };
    auto cost = [&](uint32_t e) { return cost_of(a, e, pre_lo, pre_hi); };
    bool falls = false;
    auto scan = [&](uint32_t v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= (uint32_t)o) v += u;
        }
        return v;
    };
    const bool with_pre = n_entries > c.n_seqs;
    if (n_entries <= kFew) {
        if (with_pre) {
            seen_of(a, lane, 32, pre_lo, pre_hi);
            pre_lo = __reduce_min_sync(0xffffffffu, pre_lo);
            pre_hi = __reduce_max_sync(0xffffffffu, pre_hi);
        }
        // (not unrolled: what a warp runs once costs most where its instructions come from)
        uint32_t v = 0;
#pragma unroll 1
        for (uint32_t k = 0; k < n_entries; k += 32) {
            v = k + lane < n_entries ? cost_of(a, k + lane, pre_lo, pre_hi, falls) : 0;
            costs[warp][k + lane] = v;
            total += __reduce_add_sync(0xffffffffu, v);
        }
        falls = __any_sync(0xffffffffu, falls);
        share();
        uint32_t at = 0;
#pragma unroll 1
        for (uint32_t k = 0; k < n_entries; k += 32) {
            if (n_entries > 32) v = costs[warp][k + lane];
            const uint32_t inc = scan(v) + at;
            if (n_entries > kFewMerged && blockIdx.x == 0 && warp == 0 && k + lane < n_entries) a.plan[kPlanHead + k + lane] = inc - v;
            const uint32_t here = __ballot_sync(0xffffffffu, v && x0 >= inc - v && x0 < inc);
            if (here) {
                e_first = k + __ffs(here) - 1;
                e_before = __shfl_sync(0xffffffffu, inc - v, __ffs(here) - 1);
            }
            at = __shfl_sync(0xffffffffu, inc, 31);
        }
    } else {
        if (with_pre) {
            seen_of(a, tid, kWarps * 32, pre_lo, pre_hi);
            atomicMin(&edge[0], pre_lo);
            atomicMax(&edge[1], pre_hi);
            __syncthreads();
            pre_lo = edge[0];
            pre_hi = edge[1];
        }
        const uint32_t per = (n_entries + kWarps * 32 - 1) / (kWarps * 32), beg = min(n_entries, tid * per), end = min(n_entries, beg + per);
        uint32_t sum = 0;
        for (uint32_t e = beg; e < end; e++) {
            before[e] = sum;
            sum += cost_of(a, e, pre_lo, pre_hi, falls);
        }
        const uint32_t inc = scan(sum);
        if (lane == 31) sums[warp] = inc;
        __syncthreads();
        uint32_t off = inc - sum;
        for (uint32_t w = 0; w < warp; w++) off += sums[w];
        for (uint32_t e = beg; e < end; e++) {
            before[e] += off;
            if (blockIdx.x == 0) a.plan[kPlanHead + e] = before[e];
        }
        if (tid == kWarps * 32 - 1) before[n_entries] = off + sum;
        falls = __syncthreads_or(falls);
        total = before[n_entries];
        share();
        uint32_t l = 0, r = n_entries;         // the last entry that begins at or before x0 (those without steps come before it)
        while (r - l > 1) {
            const uint32_t mid = (l + r) / 2;
            if (before[mid] <= x0) l = mid;
            else r = mid;
        }
        e_first = l;
        e_before = before[l];
    }
    if (n_entries > kFewMerged && blockIdx.x == 0 && tid == 0) {
        a.plan[0] = pre_lo;
        a.plan[1] = pre_hi;
        a.plan[2] = falls ? 0 : total;
        a.plan[3] = workers;
    }
    if (x0 == x1 || falls) return;             // (a count of 0 instead took 6 more registers, and 2.4 us of 131072 positions)

    // A place in the order of steps.  Reader and copier walk it, the copier kStages ahead.
    struct Cursor {
        Entry t;
        uint32_t e, h, tile, lo, hi, step;     // lo, hi: positions that the tile's rows see
    };
    auto enter = [&](Cursor& u) {              // (e, h, tile) are set
        u.lo = u.t.lo;
        u.hi = u.t.hi;
        if (u.e < c.n_seqs && u.t.tiles > 1) {
            const uint32_t last = min(u.t.n * c.group, (u.tile + 1) * kRows) - 1;
            const int32_t p0 = u.t.base + (int32_t)(u.tile * kRows / c.group), p1 = u.t.base + (int32_t)(last / c.group);
            u.hi = (uint32_t)max(0, p1 + 1);
            u.lo = max(u.lo, first_seen(p0, a.window));
        }
    };
    auto next = [&](Cursor& u, uint32_t x) {   // to step x, the one behind
        if (++u.step < u.t.steps) return;
        u.step = 0;
        if (++u.tile == u.t.tiles) {
            u.tile = 0;
            if (++u.h == c.kv_heads) {
                u.h = 0;
                if (x >= total) return;
                uint32_t some = 0;             // the next entry that has steps (there is one)
                for (u.e++; !(some = __ballot_sync(0xffffffffu, u.e + lane < n_entries && cost(u.e + lane))) && u.e < n_entries; u.e += 32) {}
                u.e += __ffs(some) - 1;
                u.t = entry_of(a, u.e, pre_lo, pre_hi);
            }
        }
        enter(u);
    };
    auto key_of = [&](const Cursor& u) { return (u.t.lo & ~(kBox - 1)) + u.step * kStep; };
    auto hidden = [&](const Cursor& u) { return key_of(u) >= u.hi || key_of(u) + kStep <= u.lo; };      // from all rows of the tile

    const uint32_t bar0 = smem_u32(&bars[warp * S::kStages]), ring0 = smem_u32(ring) + warp * S::kStages * S::kStage;
    Cursor in, at;
    at.e = e_first;
    at.t = entry_of(a, at.e, pre_lo, pre_hi);
    {
        const uint32_t of = x0 - e_before, seg = of / at.t.steps;
        at.h = seg / at.t.tiles;
        at.tile = seg % at.t.tiles;
        at.step = of % at.t.steps;
        enter(at);
    }
    in = at;
    // pages of the next 32 boxes of the copier's segment, one a lane
    int32_t pages = 0;
    uint32_t pages_at = 0;                     // the step whose boxes come first
    auto look_up = [&]() {
        const uint32_t k = key_of(in) + lane * kBox;
        pages = k < in.hi ? in.t.table[k >> c.page_log2] : 0;
        pages_at = in.step;
    };
    auto advance = [&](uint32_t x) {
        next(in, x);
        if (in.step == 0 || in.step == pages_at + 16) look_up();
    };
    auto copy = [&](uint32_t stage) {
        const uint32_t k = key_of(in), n = hidden(in) ? 0 : k + kBox < in.hi ? 2 : 1;
        int32_t page[2];
#pragma unroll
        for (uint32_t b = 0; b < 2; b++) {
            page[b] = __shfl_sync(0xffffffffu, pages, 2 * (in.step - pages_at) + b);
            if (b < n && (uint32_t)page[b] >= c.n_pages) {
                report(c);
                page[b] = 0;
            }
        }
        if (lane == 0) {
            const uint32_t bar = bar0 + 8 * stage, dst = ring0 + stage * S::kStage;
            mbar_expect_tx(bar, n * 2 * S::kBoxBytes);
#pragma unroll
            for (uint32_t b = 0; b < 2; b++) {
                if (b >= n) break;
                const uint32_t p = k + b * kBox;
                const int32_t row = (int32_t)((((uint32_t)page[b] * c.kv_heads + in.h) << c.page_log2) + (p & ((1u << c.page_log2) - 1)));
                tma_load_3d(dst + b * S::kBoxBytes, &mk, 0, row, 0, bar);
                tma_load_3d(dst + (2 + b) * S::kBoxBytes, &mv, 0, row, 0, bar);
            }
        }
        __syncwarp();
    };
    uint32_t xin = x0;
    look_up();

    uint32_t qa[KS][4], lo[2], hi[2];
    int32_t pos[2];
    size_t orow[2];                            // (row, head) of a thread's two rows
    bool live[2];
    float o[ND][4], m[2], l[2];
    // scores times mul are in units of log2; plain: products are scores times a positive scale.  Else they are scaled (before the cap or here) and biased.
    const bool plain = a.cap == 0.f && !a.slopes && a.scale > 0.f;
    const float mul = plain ? a.scale * kLog2e : kLog2e, pre = a.cap != 0.f ? a.cap : a.scale;
    float slope[2];
    auto begin = [&]() {                       // rows of the reader's segment
#pragma unroll
        for (uint32_t r = 0; r < 2; r++) {
            const uint32_t i = at.tile * kRows + g4 + 8 * r;
            live[r] = i < at.t.n * c.group;
            const uint32_t nth = at.t.n > 1 ? i / c.group : 0;   // (a division costs more than the rest of this)
            const uint32_t token = at.t.row0 + (live[r] ? nth : 0), head = at.h * c.group + (live[r] ? i - nth * c.group : 0);
            pos[r] = at.t.base + (int32_t)nth;
            uint32_t limit = 0x7FFFFFFFu;
            if (at.e >= c.n_seqs && live[r]) {
                const uint32_t s = sequence_by_halves(c, token);
                live[r] = s < c.n_seqs;
                if (live[r]) {
                    const Seq q = sequence(c, s);
                    live[r] = token >= q.row0 && token < q.row0 + q.n;
                    pos[r] = (int32_t)q.len - (int32_t)(q.row0 + q.n - token);
                }
                limit = c.shared;
            }
            orow[r] = (size_t)token * c.heads + head;
            lo[r] = live[r] ? first_seen(pos[r], a.window) : 0;
            if (live[r] && at.e < c.n_seqs) lo[r] = max(lo[r], c.shared);
            hi[r] = live[r] ? min((uint32_t)max(0, pos[r] + 1), limit) : 0x7FFFFFFFu;
            slope[r] = a.slopes && live[r] ? a.slopes[head] : 0.f;
            const uint32_t* qp = reinterpret_cast<const uint32_t*>(reinterpret_cast<const T*>(a.q) + (size_t)token * a.ldq + (size_t)head * HD);
#pragma unroll
            for (uint32_t k = 0; k < KS; k++) {
                qa[k][r] = live[r] ? qp[8 * k + t4] : 0;
                qa[k][2 + r] = live[r] ? qp[8 * k + 4 + t4] : 0;
            }
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
#pragma unroll
        for (uint32_t d = 0; d < ND; d++) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
    };
    // `whole`: this worker has had all steps of the segment
    auto finish = [&](bool whole, bool first) {
#pragma unroll
        for (uint32_t r = 0; r < 2; r++) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (!live[r]) continue;
            if (whole && c.shared == 0) {
                const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
                uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(a.out) + orow[r] / c.heads * a.ldo + orow[r] % c.heads * HD);
#pragma unroll
                for (uint32_t d = 0; d < ND; d++) dst[4 * d + t4] = Half2<T>::pack(o[d][2 * r] * inv, o[d][2 * r + 1] * inv);
                continue;
            }
            float *po, *pml;
            if (whole) {
                const bool pre = at.e >= c.n_seqs;
                po = (pre ? a.pre_o : a.row_o) + orow[r] * HD;
                pml = (pre ? a.pre_ml : a.row_ml) + orow[r] * 2;
            } else {
                const Piece p = slot_of(a, me, first);
                po = p.o + (g4 + 8 * r) * HD;
                pml = p.ml + (g4 + 8 * r) * 2;
            }
#pragma unroll
            for (uint32_t d = 0; d < ND; d++) *reinterpret_cast<float2*>(po + 8 * d + 2 * t4) = make_float2(o[d][2 * r], o[d][2 * r + 1]);
            if (t4 == 0) *reinterpret_cast<float2*>(pml) = make_float2(m[r] - Half2<T>::kLift, l[r]);      // what the sums are relative to
        }
    };

    bool ok = true;
    uint32_t begun = x0 - at.step;             // where the segment begins in the order of steps
    for (uint32_t s = 0; s < S::kStages && xin < x1; s++) {
        copy(s);
        xin++;
        if (xin < x1) advance(xin);
    }
    begin();
    for (uint32_t x = x0; x < x1 && ok; x++) {
        const uint32_t n = x - x0, stage = n % S::kStages;
        ok = __all_sync(0xffffffffu, mbar_wait(bar0 + 8 * stage, (n / S::kStages) & 1));
        if (!ok) break;
        const uint32_t k0 = key_of(at);
        if (!hidden(at)) {
            const uint32_t sk = ring0 + stage * S::kStage, sv = sk + 2 * S::kBoxBytes;
            float s[NK][4];
            uint32_t row_at[NK];                   // a lane's place among the rows of keys 8 j .. 8 j + 7
#pragma unroll
            for (uint32_t j = 0; j < NK; j++) {
                s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
                row_at[j] = sk + (j >> 1) * S::kBoxBytes + ((j & 1) * 8 + (lane & 7)) * 128;
            }
            // products of four blocks of keys next to each other, none of which waits for another
            uint32_t b[2][NK][4];
            auto keys = [&](uint32_t k, uint32_t (&x)[NK][4]) {
                const uint32_t ch = 2 * k + (lane >> 3);                            // 16-byte piece of the key's row
#pragma unroll
                for (uint32_t j = 0; j < NK; j++) ldsm_x4(x[j], row_at[j] + (ch >> 3) * (kBox * 128) + (((ch & 7) ^ (lane & 7)) << 4));
            };
            keys(0, b[0]);
#pragma unroll
            for (uint32_t k = 0; k < KS; k += 2) {
                if (k + 2 < KS) keys(k + 2, b[(k / 2 + 1) & 1]);
#pragma unroll
                for (uint32_t j = 0; j < NK; j++) Half2<T>::mma(s[j], qa[k], b[(k / 2) & 1][j][0], b[(k / 2) & 1][j][1]);
#pragma unroll
                for (uint32_t j = 0; j < NK; j++) Half2<T>::mma(s[j], qa[k + 1], b[(k / 2) & 1][j][2], b[(k / 2) & 1][j][3]);
            }
            // a thread has keys 8 j + 2 t4, + 1 of rows g4 and g4 + 8
            const bool inside = k0 >= lo[0] && k0 >= lo[1] && k0 + kStep <= hi[0] && k0 + kStep <= hi[1];
            const bool all = __all_sync(0xffffffffu, inside);
            float top[2] = {-INFINITY, -INFINITY};
            if (!plain || !all) {
                if (a.cap != 0.f) tanh_scores(reinterpret_cast<float(&)[4 * NK]>(s), a.tanh);
                // in units of mul afterwards, like the plain ones
#pragma unroll
                for (uint32_t j = 0; j < NK; j++)
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++) {
                        const uint32_t r = e >> 1, key = k0 + 8 * j + 2 * t4 + (e & 1);
                        float v = plain ? s[j][e] : s[j][e] * pre - slope[r] * (float)(pos[r] - (int32_t)key);
                        if (key < lo[r] || key >= hi[r]) v = -INFINITY;
                        s[j][e] = v;
                    }
            }
#pragma unroll
            for (uint32_t j = 0; j < NK; j++)
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) top[e >> 1] = fmaxf(top[e >> 1], s[j][e]);
            float corr[2];
            bool rise = false;
#pragma unroll
            for (uint32_t r = 0; r < 2; r++) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                top[r] *= mul;
                const float now = fmaxf(m[r], top[r]);
                corr[r] = now > m[r] ? exp2_approx(m[r] - now) : 1.f;
                rise |= now > m[r];
                m[r] = now;
                l[r] *= corr[r];
            }
            if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                for (uint32_t d = 0; d < ND; d++) {
                    o[d][0] *= corr[0];
                    o[d][1] *= corr[0];
                    o[d][2] *= corr[1];
                    o[d][3] *= corr[1];
                }
            }
            const float sub[2] = {m[0] == -INFINITY ? 0.f : m[0] - Half2<T>::kLift, m[1] == -INFINITY ? 0.f : m[1] - Half2<T>::kLift};
            // the product's rounding against that of the maximum (2^-24 of the score) stays in the weight, as an f32 score's own would
#pragma unroll
            for (uint32_t j = 0; j < NK; j++)
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    s[j][e] = exp2_approx(fmaf(s[j][e], mul, -sub[e >> 1]));
                    l[e >> 1] += s[j][e];
                }
            uint32_t bad = 0;
#pragma unroll
            for (uint32_t k = 0; k < kStep / 16; k++) {
                if (k0 + 16 * k >= at.hi) break;                // not copied
                // of the two keys in a word of V: the bits of those that some row of the tile sees
                const uint32_t ka = k0 + 16 * k + 2 * t4;
                uint32_t seen[2];
#pragma unroll
                for (uint32_t i = 0; i < 2; i++)
                    seen[i] = (ka + 8 * i >= at.lo && ka + 8 * i < at.hi ? 0x8000u : 0) | (ka + 8 * i + 1 >= at.lo && ka + 8 * i + 1 < at.hi ? 0x80000000u : 0);
                // the weights meet the values in the cache's type: half a step of it, relative, each (Half2: how far down); their sum is that of the 32-bit ones
                const uint32_t pa[4] = {Half2<T>::pack(s[2 * k][0], s[2 * k][1]), Half2<T>::pack(s[2 * k][2], s[2 * k][3]), Half2<T>::pack(s[2 * k + 1][0], s[2 * k + 1][1]),
                                        Half2<T>::pack(s[2 * k + 1][2], s[2 * k + 1][3])};
                const uint32_t row = ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
                for (uint32_t d = 0; d < ND; d += 2) {
                    uint32_t b[4];
                    const uint32_t ch = d + (lane >> 4);
                    ldsm_x4_trans(b, sv + k * S::kBoxBytes + (ch >> 3) * (kBox * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
                    if (!all) {                // a hidden position's weight of 0 would meet whatever lies there, and 0 x Inf is NaN
#pragma unroll
                        for (uint32_t i = 0; i < 4; i++) {
                            const uint32_t nf = Half2<T>::not_finite(b[i]);
                            b[i] = finite_part<T>(b[i], nf);
                            bad |= nf & seen[i & 1];
                        }
                    }
                    Half2<T>::mma(o[d], pa, b[0], b[1]);
                    Half2<T>::mma(o[d + 1], pa, b[2], b[3]);
                }
            }
            if (!all && __any_sync(0xffffffffu, bad != 0)) {
                float x[ND][4];                // a copy: what a call is given by address lives in memory from beginning to end
#pragma unroll
                for (uint32_t d = 0; d < ND; d++) x[d][0] = o[d][0], x[d][1] = o[d][1], x[d][2] = o[d][2], x[d][3] = o[d][3];
                float y[NK][4];
#pragma unroll
                for (uint32_t j = 0; j < NK; j++) y[j][0] = s[j][0], y[j][1] = s[j][1], y[j][2] = s[j][2], y[j][3] = s[j][3];
                const uint32_t from[2] = {lo[0], lo[1]}, to[2] = {hi[0], hi[1]};
                add_not_finite<T, HD>(ring + warp * S::kStages * S::kStage + stage * S::kStage + 2 * S::kBoxBytes, k0, at.hi, from, to, y, x);
#pragma unroll
                for (uint32_t d = 0; d < ND; d++) o[d][0] = x[d][0], o[d][1] = x[d][1], o[d][2] = x[d][2], o[d][3] = x[d][3];
            }
        }
        __syncwarp();
        if (xin < x1) {
            copy(stage);
            xin++;
            if (xin < x1) advance(xin);
        }
        const uint32_t left = at.t.steps - at.step - 1;
        if (left == 0 || x + 1 == x1) {
            finish(left == 0 && begun >= x0, begun <= x0);
            next(at, x + 1);
            begun = x + 1;
            if (x + 1 < x1) begin();
        } else next(at, x + 1);
    }
    if (!ok) {
        mbar_drain(bar0, S::kStages, xin - x0);
        if (lane == 0 && c.status) atomicCAS(c.status, 0, 1);
    }
}

// Adds up what the launches have left of a (row, query head): a warp for each, or a block (WIDE) where a segment has many pieces.  A lane has the reference and sum
// of a piece, the factors 2^(m - max m) go round, and every lane adds up 2 or 4 of the dimensions.  Rows that a worker has written itself are left.
struct MergeArgs {
    uint32_t n_entries, most;                  // of the split kernel, and its workers at most: no entries when it has not run (all sequences, and the shared positions if their rows are few)
    uint32_t own_parts, pre_parts;             // parts of the kernel for many rows: 0 when the split kernel has had those positions
    const float *own_o, *own_ml, *pre_o, *pre_ml;
    bool shared;
};
// Sums of so many pieces are asked for at once: the registers for more of them cost warps that hide the rest (64 sequences with 1792 rows of pieces 43.9 us; with 5 44.4,
// with 8 in blocks of 8 warps 46.0).
constexpr uint32_t kMergeWarps = 4, kWideWarps = 16, kAsked = 4;

// Sequence of a row, by a warp: 33 parts at a time.
__device__ __forceinline__ uint32_t sequence_by_warp(const Cache& c, uint32_t row) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, n = c.n_seqs;             // as many of q_start[1 ..] as are <= row: lo of them, and some of the n behind
    while (n > 0) {
        const uint32_t step = n / 33 + 1, at = lo + (lane + 1) * step;
        const uint32_t hit = __popc(__ballot_sync(0xffffffffu, at <= lo + n && c.q_start[at] <= (int32_t)row));
        const uint32_t end = lo + n;
        lo += hit * step;
        n = min(step - 1, end - lo);
    }
    return lo;
}

template <typename T, int HD, bool WIDE>
__global__ void __launch_bounds__((WIDE ? kWideWarps : kMergeWarps) * 32) merge_kernel(const AttnArgs a, const MergeArgs g) {
    constexpr uint32_t E = HD / 32;
    const Cache& c = a.c;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t pairs = (uint64_t)c.rows * c.heads, orow = WIDE ? blockIdx.x : (uint64_t)blockIdx.x * kMergeWarps + warp;
    // The lengths are read ahead of the wait, which every warp does all the same, as whoever comes next relies on this launch's being the last to end.
    acquire_ahead(c);
    const uint32_t token = (uint32_t)(orow / c.heads), head = (uint32_t)(orow % c.heads);
    const uint32_t s = orow < pairs ? sequence_by_warp(c, token) : c.n_seqs;
    const Seq q = s < c.n_seqs ? sequence(c, s) : Seq{0, 0, 0};
    // the split kernel's plan, as far as it concerns this row; that of many entries it has left in the scratch
    uint32_t workers = 1, total = 0, pre_lo = c.shared, pre_hi = 0, before = 0, before_pre = 0;
    const bool mine = token >= q.row0 && token < q.row0 + q.n;
    // pieces of one entry: as many, from worker w0 on, or one that is whole
    struct List {
        uint32_t n, w0, beg, row;
    };
    auto list_of = [&](const Entry& u, uint32_t first, uint32_t i) {
        List x{0, 0, 0, i % kRows};
        if (u.steps == 0 || total == 0) return x;
        x.beg = first + (head / c.group * u.tiles + i / kRows) * u.steps;
        x.w0 = owner_of(x.beg, total, workers);
        x.n = owner_of(x.beg + u.steps - 1, total, workers) - x.w0 + 1;
        return x;
    };
    List own{g.own_parts, 0, 0, 0}, pre{g.pre_parts, 0, 0, 0};
    auto look_up = [&]() {
        own = list_of(entry_of(a, s, pre_lo, pre_hi), before, (token - q.row0) * c.group + head % c.group);
        if (g.n_entries > c.n_seqs) pre = list_of(entry_of(a, c.n_seqs, pre_lo, pre_hi), before_pre, token * c.group + head % c.group);
    };
    if (g.n_entries && g.n_entries <= kFewMerged) {
        if (g.n_entries > c.n_seqs) {
            seen_of(a, lane, 32, pre_lo, pre_hi);
            pre_lo = __reduce_min_sync(0xffffffffu, pre_lo);
            pre_hi = __reduce_max_sync(0xffffffffu, pre_hi);
        }
        bool falls = false;
#pragma unroll 1
        for (uint32_t k = lane; k < g.n_entries; k += 32) {
            const uint32_t v = cost_of(a, k, pre_lo, pre_hi, falls);
            total += v;
            if (k < s) before += v;
            if (k < c.n_seqs) before_pre += v;
        }
        total = __any_sync(0xffffffffu, falls) ? 0 : __reduce_add_sync(0xffffffffu, total);
        before = __reduce_add_sync(0xffffffffu, before);
        before_pre = __reduce_add_sync(0xffffffffu, before_pre);
        workers = workers_of(total, g.most);
        if (mine) look_up();
    }
    grid_dependency_wait();
    grid_launch_dependents();
    if (!mine) return;
    if (g.n_entries > kFewMerged) {
        pre_lo = a.plan[0];
        pre_hi = a.plan[1];
        total = a.plan[2];
        workers = a.plan[3];
        before = a.plan[kPlanHead + s];
        if (g.n_entries > c.n_seqs) before_pre = a.plan[kPlanHead + c.n_seqs];
        look_up();
    }
    if (g.n_entries && own.n == 1 && !g.shared) return;
    const uint32_t n = own.n + pre.n, step = WIDE ? kWideWarps : 1;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (uint32_t e = 0; e < E; e++) o[e] = 0.f;
    for (uint32_t i0 = WIDE ? warp : 0; i0 < n; i0 += 32 * step) {           // a warp's pieces i0, i0 + step, ...: 32 at a time
        uint32_t i = i0 + lane * step;
        const uint32_t count = min(32u, (n - i0 + step - 1) / step);
        const float *po = a.slot_o, *pml = nullptr;
        if (i < n) {
            const bool p = i >= own.n;
            const List& x = p ? pre : own;
            if (p) i -= own.n;
            if (p ? g.pre_parts : g.own_parts) {
                po = (p ? g.pre_o : g.own_o) + (i * pairs + orow) * HD;
                pml = (p ? g.pre_ml : g.own_ml) + (i * pairs + orow) * 2;
            } else if (x.n == 1) {
                po = (p ? a.pre_o : a.row_o) + orow * HD;
                pml = (p ? a.pre_ml : a.row_ml) + orow * 2;
            } else {
                const Piece y = slot_of(a, x.w0 + i, begin_of(x.w0 + i, total, workers) >= x.beg);
                po = y.o + x.row * HD;
                pml = y.ml + x.row * 2;
            }
        }
        // the sums of the first ones are asked for along with the maxima
        const uint64_t at = reinterpret_cast<uint64_t>(po);
        float v[kAsked][E];
        auto ask = [&](uint32_t k, float (&x)[E]) {
            const float* y = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, at, k & 31));
            if (k >= count) return;
            if constexpr (E == 4) {
                const float4 z = *reinterpret_cast<const float4*>(y + 4 * lane);
                x[0] = z.x; x[1] = z.y; x[2] = z.z; x[3] = z.w;
            } else {
                const float2 z = *reinterpret_cast<const float2*>(y + 2 * lane);
                x[0] = z.x; x[1] = z.y;
            }
        };
#pragma unroll
        for (uint32_t k = 0; k < kAsked; k++) ask(k, v[k]);
        const float2 ml = pml ? *reinterpret_cast<const float2*>(pml) : make_float2(-INFINITY, 0.f);
        float top = fmaxf(m, ml.x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        // no score at all: the sums are 0, or no numbers
        const float f = !pml ? 0.f : top == -INFINITY ? 1.f : exp2_approx(ml.x - top), old = top == -INFINITY ? 1.f : exp2_approx(m - top);
        float sum = pml ? f * ml.y : 0.f;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        l = fmaf(l, old, sum);
        m = top;
#pragma unroll
        for (uint32_t e = 0; e < E; e++) o[e] *= old;
        for (uint32_t k0 = 0; k0 < count; k0 += kAsked) {
#pragma unroll
            for (uint32_t k = 0; k < kAsked; k++) {
                const float fk = __shfl_sync(0xffffffffu, f, (k0 + k) & 31);
                if (k0 + k >= count) continue;
#pragma unroll
                for (uint32_t e = 0; e < E; e++) o[e] = fmaf(fk, v[k][e], o[e]);
            }
            if (k0 + kAsked < count)
#pragma unroll
                for (uint32_t k = 0; k < kAsked; k++) ask(k0 + kAsked + k, v[k]);
        }
    }
    if constexpr (WIDE) {
        __shared__ float sm[kWideWarps], sl[kWideWarps], so[kWideWarps][HD];
        if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
        for (uint32_t e = 0; e < E; e++) so[warp][E * lane + e] = o[e];
        __syncthreads();
        if (warp > 0) return;
        float top = m;
#pragma unroll
        for (uint32_t w = 1; w < kWideWarps; w++) top = fmaxf(top, sm[w]);
        l = 0.f;
#pragma unroll
        for (uint32_t e = 0; e < E; e++) o[e] = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kWideWarps; w++) {
            const float f = top == -INFINITY ? 1.f : exp2_approx(sm[w] - top);
            l = fmaf(f, sl[w], l);
#pragma unroll
            for (uint32_t e = 0; e < E; e++) o[e] = fmaf(f, so[w][E * lane + e], o[e]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(a.out) + (size_t)token * a.ldo + (size_t)head * HD);
#pragma unroll
    for (uint32_t e = 0; e < E / 2; e++) dst[lane * (E / 2) + e] = Half2<T>::pack(o[2 * e] * inv, o[2 * e + 1] * inv);
}

// ── which kernel has which positions, and the scratch ──
// By the (row, query head) pairs that share keys: up to 16 (a tile of the split kernel) it is bound by the copies, beyond that it reads its keys again for every
// 16, from the second-level cache.  Where that makes fewer than eight steps a worker, it is done before a launch of the other kernel would be: 40 pairs behind 9216
// positions 13 us and 21, 238 behind 384 with 4 key heads 14 and 20; at 18 steps a worker (288 pairs behind 18816) it is 37 and 29.  (Rows of a sequence's
// own go to the other kernel from 32 pairs on, however few: 45 rows 12 us and 19.)  The parts of the kernel for many rows: as many as take the least time, which is that of a part (its blocks, and four more for what it takes to begin and to
// end) as often as the parts go round 148 SMs, a tenth of a block a part for the sums, and five blocks for the merge where there is none with one part.
// (40 pairs behind 9216 shared positions: 18 parts 21 us, one 131; 288 behind 18816: 29 parts 29 us, 25 of them 34; two prompts of 700 rows behind a window
// of 143, 16 heads: one part 25 us, three 59; 250 rows, 32 heads, without anything in front: one part 16 us, two 22.)
struct Choice {
    bool own_tc, pre_tc, direct;
    uint32_t own_tiles, pre_tiles, own_split, pre_split, n_entries;
};
static uint32_t parts_of(uint64_t ctas, uint64_t blocks, double apart) {
    uint32_t best = 1;
    double least = 1e30;
    for (uint32_t z = 1; z <= 64 && (z == 1 || z <= blocks); z++) {
        const double took = (double)((ctas * z + 147) / 148) * (double)((blocks + z - 1) / z + 4) + 0.1 * z + (z > 1 ? apart : 0.0);
        if (took < least) {
            least = took;
            best = z;
        }
    }
    return best;
}
static Choice choose(const runit_paged_cfg* g, const runit_paged_batch* b) {
    const uint64_t group = g->heads / g->kv_heads, pairs = b->rows * group;
    Choice c;
    c.own_tc = pairs > 32ull * b->n_seqs;
    const uint64_t pre_steps = (pairs + 15) / 16 * g->kv_heads * (b->shared_len / kStep);
    c.pre_tc = b->shared_len && pairs > 16 && (c.own_tc || pre_steps > 8ull * kWarps * 148);
    c.own_tiles = (uint32_t)(pairs / 256 + b->n_seqs);
    c.pre_tiles = (uint32_t)((pairs + 255) / 256);
    const uint64_t all = (uint64_t)b->table_ld * g->page, seen = g->window ? min(all, (uint64_t)g->window + 256) : all;
    c.own_split = parts_of((pairs / 256 + (b->n_seqs + 1) / 2) * g->kv_heads, (seen + 127) / 128, b->shared_len ? 0.0 : 5.0);
    c.pre_split = parts_of((uint64_t)c.pre_tiles * g->kv_heads, b->shared_len / 128, 0.0);
    c.direct = c.own_tc && !b->shared_len && c.own_split == 1;
    c.n_entries = c.own_tc ? 0 : b->n_seqs + (b->shared_len && !c.pre_tc ? 1 : 0);       // (own_tc: more than 32 pairs, so pre_tc as well)
    return c;
}
struct Layout {
    size_t plan, slot_o, slot_ml, row_o, row_ml, pre_o, pre_ml, own_part_o, own_part_ml, pre_part_o, pre_part_ml, bytes;
};
static Layout layout_of(const runit_paged_cfg* g, const runit_paged_batch* b, const Choice& c) {
    Layout l;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t p = at;
        at += (n + 255) & ~(size_t)255;
        return p;
    };
    const size_t pairs = (size_t)b->rows * g->heads, row = b->shared_len && !c.own_tc ? pairs : 0, pre = b->shared_len && !c.pre_tc ? pairs : 0;
    const size_t slots = c.n_entries ? 2 * (size_t)kMaxWorkers * kRows : 0, own_parts = c.own_tc && !c.direct ? c.own_split * pairs : 0, pre_parts = c.pre_tc ? c.pre_split * pairs : 0;
    l.plan = take((kPlanHead + kMaxSeqs + 2) * 4);
    l.slot_o = take(slots * g->dim * 4);
    l.slot_ml = take(slots * 8);
    l.row_o = take(row * g->dim * 4);
    l.row_ml = take(row * 8);
    l.pre_o = take(pre * g->dim * 4);
    l.pre_ml = take(pre * 8);
    l.own_part_o = take(own_parts * g->dim * 4);
    l.own_part_ml = take(own_parts * 8);
    l.pre_part_o = take(pre_parts * g->dim * 4);
    l.pre_part_ml = take(pre_parts * 8);
    l.bytes = at;
    return l;
}

static int32_t encode(runit_ctx* ctx, const runit_paged_cfg* g, void* pages, CUtensorMap* m) {
    if (!ctx->encode_tiled) return runit_fail(ctx, RUNIT_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled is not available");
    auto f = reinterpret_cast<CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                           const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill)>(ctx->encode_tiled);
    const cuuint64_t dim[3] = {64, (cuuint64_t)g->n_pages * g->kv_heads * g->page, g->dim / 64}, stride[2] = {g->dim * 2ull, 128};
    const cuuint32_t box[3] = {64, kBox, g->dim / 64}, one[3] = {1, 1, 1};
    const CUresult r = f(m, g->type == RUNIT_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, pages, dim, stride, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return runit_fail(ctx, RUNIT_ERR_LAUNCH, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return RUNIT_OK;
}

template <typename T, int HD>
static int32_t run(runit_ctx* ctx, const runit_paged_cfg* g, const runit_paged_batch* b, const AttnArgs& a, const Choice& c, uint8_t* s, const Layout& l) {
    int32_t st;
    TcArgs pre{min(g->page, 128u), c.pre_split, true, false, false, (float*)(s + l.pre_part_o), (float*)(s + l.pre_part_ml)};
    TcArgs own{min(g->page, 128u), c.own_split, false, c.direct, false, (float*)(s + l.own_part_o), (float*)(s + l.own_part_ml)};
    uint32_t share = 0, most = 0;
    if (c.n_entries) {
        constexpr uint32_t smem = Shape<HD>::kRing + 1024 + (kMaxSeqs + 2) * 4;
        static bool configured[64] = {false};
        if (ctx->device >= 64 || !configured[ctx->device]) {
            RUNIT_CUDA_TRY(ctx, cudaFuncSetAttribute(paged_split_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            if (ctx->device < 64) configured[ctx->device] = true;
        }
        CUtensorMap mk, mv;
        if ((st = encode(ctx, g, g->k_pages, &mk)) != RUNIT_OK || (st = encode(ctx, g, g->v_pages, &mv)) != RUNIT_OK) return st;
        const uint32_t grid = min((uint32_t)ctx->sm_count, kMaxWorkers / kWarps);
        runit_launch_chain_smem(ctx, paged_split_kernel<T, HD>, dim3(grid), dim3(kWarps * 32), smem, mk, mv, a, c.n_entries);
        if ((st = runit_after_launch(ctx, "paged_attention")) != RUNIT_OK) return st;
        most = grid * kWarps;
        share = most / (c.n_entries * g->kv_heads);
    }
    // A launch behind another one of this call reads nothing of it, and takes the SMs that it leaves: 128 rows behind 32768 positions 120 -> 115 us.  Only the
    // second one: its own successor could not rely on its having waited.
    pre.beside = c.n_entries > 0;
    own.beside = c.pre_tc;                     // the split kernel has not run
    if (c.pre_tc && (st = paged_attention_tc(ctx, g, a, pre, c.pre_tiles)) != RUNIT_OK) return st;
    if (c.own_tc && (st = paged_attention_tc(ctx, g, a, own, c.own_tiles)) != RUNIT_OK) return st;
    if (c.direct) return RUNIT_OK;
    const MergeArgs m{c.n_entries, most, c.own_tc ? c.own_split : 0, c.pre_tc ? c.pre_split : 0, own.part_o, own.part_ml, pre.part_o, pre.part_ml, b->shared_len != 0};
    // a block for each where a segment has more pieces than a warp asks for at once, when all are alike
    const uint64_t pairs = (uint64_t)g->heads * b->rows;
    if (share >= 16) runit_launch_chain(ctx, merge_kernel<T, HD, true>, dim3((uint32_t)pairs), dim3(kWideWarps * 32), a, m);
    else runit_launch_chain(ctx, merge_kernel<T, HD, false>, dim3((uint32_t)((pairs + kMergeWarps - 1) / kMergeWarps)), dim3(kMergeWarps * 32), a, m);
    return runit_after_launch(ctx, "paged_attention (merge)");
}

}  // namespace pg
}  // namespace runit

using namespace runit;

extern "C" {

size_t runit_paged_attention_scratch_bytes(const runit_paged_cfg* cfg, const runit_paged_batch* batch) {
    return pg::why_not(cfg, batch) ? 0 : pg::layout_of(cfg, batch, pg::choose(cfg, batch)).bytes;
}

int32_t runit_paged_attention(runit_ctx_t* ctx, const runit_paged_cfg* cfg, const runit_paged_batch* batch, const void* q, uint32_t ldq, void* out,
                              uint32_t ldo, void* scratch, size_t scratch_bytes) {
    if (!ctx) return RUNIT_ERR_BAD_ARG;
    const char* why = pg::why_not(cfg, batch);
    if (!why) why = pg::why_not_memory(cfg, batch);
    RUNIT_REQUIRE(ctx, !why, "paged_attention: %s", why);
    RUNIT_REQUIRE(ctx, q && out && runit_aligned(q, 16) && runit_aligned(out, 16), "paged_attention: q and out must be 16-byte aligned");
    RUNIT_REQUIRE(ctx, q != out, "paged_attention: q is read by several workers and must not be out");
    RUNIT_REQUIRE(ctx, ldq % 8 == 0 && ldo % 8 == 0 && ldq >= (uint64_t)cfg->heads * cfg->dim && ldo >= (uint64_t)cfg->heads * cfg->dim,
                  "paged_attention: ldq=%u, ldo=%u must be multiples of 8, rows of heads * dim at least", ldq, ldo);
    RUNIT_REQUIRE(ctx, scratch && runit_aligned(scratch, 256), "paged_attention: scratch must be 256-byte aligned");
    const pg::Choice c = pg::choose(cfg, batch);
    const pg::Layout l = pg::layout_of(cfg, batch, c);
    if (scratch_bytes < l.bytes) return runit_fail(ctx, RUNIT_ERR_BUFFER_SIZE, "paged_attention: %zu bytes of scratch, %zu needed", scratch_bytes, l.bytes);
    uint8_t* const s = (uint8_t*)scratch;
    const pg::AttnArgs a{pg::cache_of(ctx, cfg, batch), q, out, (const float*)cfg->slopes, ldq, ldo, cfg->window, cfg->scale, cfg->cap, pg::tanh_of(cfg->cap != 0.f ? cfg->scale / cfg->cap : 0.f), (uint32_t*)(s + l.plan),
                         (float*)(s + l.slot_o), (float*)(s + l.slot_ml), (float*)(s + l.row_o), (float*)(s + l.row_ml), (float*)(s + l.pre_o), (float*)(s + l.pre_ml)};
    if (cfg->type == RUNIT_TYPE_F16) return cfg->dim == 128 ? pg::run<__half, 128>(ctx, cfg, batch, a, c, s, l) : pg::run<__half, 64>(ctx, cfg, batch, a, c, s, l);
    return cfg->dim == 128 ? pg::run<__nv_bfloat16, 128>(ctx, cfg, batch, a, c, s, l) : pg::run<__nv_bfloat16, 64>(ctx, cfg, batch, a, c, s, l);
}

}  // extern "C"
