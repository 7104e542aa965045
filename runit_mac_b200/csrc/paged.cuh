// What the operators over a paged cache share (paged_append.cu, paged_attention.cu): the description of the cache and of a batch as the kernels
// take it, the checks of both, and the way from a row to its sequence and from a position to its page.
//
// Lengths and pages are device memory, which the host cannot check: the kernels clamp what they read there to what the tensors hold, and set
// the context's status word (code 5) where something had to be clamped.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "runit_internal.h"

namespace runit {
namespace pg {

constexpr uint32_t kMaxSeqs = 4096;

struct Cache {
    void *k, *v;
    const int32_t *table, *q_start, *kv_len;
    int32_t* status;
    uint32_t* told;                             // device word: the status has been set
    uint32_t heads, kv_heads, group, dim;       // group: query heads per key head
    uint32_t page_log2, n_pages, table_ld, n_seqs, rows, shared;
};

// The status word is host memory, which takes an atomic from the device every 0.85 us: one thread writes it, however many find something (a table of bad pages under
// 16 sequences of 8000 positions, 8 key heads, took 1.7 s, now 0.12 ms).
__device__ __forceinline__ void report(const Cache& c) {
    if (*reinterpret_cast<const volatile uint32_t*>(c.told) == 0 && atomicExch(c.told, 1u) == 0) atomicCAS(c.status, 0, 5);
}
// By every thread of a launch that reads what came before its call without having waited for the launch in front of it, which belongs to the call and has let it
// begin behind its own wait.  So whatever came before has ended and is in the second-level cache; an acquiring load sees to it that nothing read behind it
// comes from a copy that the SM has kept since earlier (the wait would do so, too).
__device__ __forceinline__ void acquire_ahead(const Cache& c) {
    int32_t first;
    asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(first) : "l"(c.q_start) : "memory");
}
// Element offset of row `pos % page` of key head h in the page of position pos; table: the sequence's pages.  A page outside the pool is
// reported and page 0 taken instead, for whoever only reads; *ok says so.
__device__ __forceinline__ size_t page_row(const Cache& c, const int32_t* table, uint32_t pos, uint32_t h, bool* ok) {
    int32_t page = table[pos >> c.page_log2];
    *ok = (uint32_t)page < c.n_pages;
    if (!*ok) {
        report(c);
        page = 0;
    }
    return ((((size_t)page * c.kv_heads + h) << c.page_log2) + (pos & ((1u << c.page_log2) - 1))) * c.dim;
}
// Rows and length of a sequence, within the tensors.  A sequence without rows is not looked at further.
struct Seq {
    uint32_t row0, n, len;
    int32_t given;                              // the length as it stands there
    bool falls;                                 // its rows would end before they begin, so that others overlap
};
__device__ __forceinline__ Seq sequence(const Cache& c, uint32_t s) {
    const int32_t a = c.q_start[s], b = c.q_start[s + 1], n = c.kv_len[s], cap = (int32_t)min((uint64_t)c.table_ld << c.page_log2, (uint64_t)0x7FFFFFFF);
    Seq q;
    q.row0 = (uint32_t)max(0, min(a, (int32_t)c.rows));
    const uint32_t end = (uint32_t)max(0, min(b, (int32_t)c.rows));
    q.n = end > q.row0 ? end - q.row0 : 0;
    q.len = (uint32_t)max(0, min(n, cap));
    q.given = n;
    q.falls = b < a;
    if (a < 0 || b < a || (uint32_t)b > c.rows || (q.n > 0 && (n < (int32_t)q.n || n > cap))) report(c);
    return q;
}

static inline const char* why_not(const runit_paged_cfg* g, const runit_paged_batch* b) {
    if (!g || !b) return "null description";
    if (g->type != RUNIT_TYPE_F16 && g->type != RUNIT_TYPE_BF16) return "the cache is f16 or bf16";
    if (g->heads == 0 || g->kv_heads == 0 || g->heads % g->kv_heads != 0 || g->heads > 1024) return "heads must be a multiple of kv_heads, at most 1024";
    if (g->dim != 64 && g->dim != 128) return "dim must be 64 or 128";
    if (g->page < 16 || g->page > 256 || (g->page & (g->page - 1)) != 0) return "page must be a power of two from 16 to 256";
    if (g->n_pages == 0 || g->n_pages > 0x7FFFFFFFu || (uint64_t)g->n_pages * g->kv_heads * g->page > 0x7FFFFFFFull) return "n_pages * kv_heads * page must be from 1 to 2^31 - 1";
    if (!std::isfinite(g->scale) || !std::isfinite(g->cap) || g->cap < 0.f) return "scale and cap must be finite, cap not negative";
    if (g->cap != 0.f && !std::isfinite(g->scale / g->cap)) return "cap is too small for the scale";
    if (b->n_seqs == 0 || b->n_seqs > kMaxSeqs) return "n_seqs must be from 1 to 4096";
    if (b->rows == 0 || (uint64_t)b->rows * g->heads > 0x7FFFFFFFull) return "rows must not be 0, and rows * heads below 2^31";
    if (b->table_ld == 0 || (uint64_t)b->table_ld * g->page > 0x7FFFFFFFull) return "table_ld must not be 0, and table_ld * page below 2^31";
    if (b->shared_len % g->page != 0 || b->shared_len / g->page > b->table_ld) return "shared_len must be whole pages, as many as a table row has at most";
    // steps of 16 positions and 16 (row, query head) pairs of a key head, all sequences together, are counted in 32 bits
    const uint64_t tiles = (uint64_t)b->rows * (g->heads / g->kv_heads) / 16 + b->n_seqs + 1, steps = (uint64_t)b->table_ld * g->page / 16 + 1;
    if (tiles * g->kv_heads >= 1ull << 32 || tiles * g->kv_heads * steps >= 1ull << 32) return "rows, sequences and table_ld * page are too many together";
    return nullptr;
}
static inline const char* why_not_memory(const runit_paged_cfg* g, const runit_paged_batch* b) {
    if (!g->k_pages || !g->v_pages || !b->table || !b->q_start || !b->kv_len) return "null pages, table, q_start or kv_len";
    if (!runit_aligned(g->k_pages, 128) || !runit_aligned(g->v_pages, 128)) return "pages must be 128-byte aligned";
    if (!runit_aligned(b->table, 4) || !runit_aligned(b->q_start, 4) || !runit_aligned(b->kv_len, 4) || !runit_aligned(g->slopes, 4)) return "table, q_start, kv_len and slopes must be 4-byte aligned";
    return nullptr;
}
static inline Cache cache_of(const runit_ctx* ctx, const runit_paged_cfg* g, const runit_paged_batch* b) {
    Cache c;
    c.k = g->k_pages;
    c.v = g->v_pages;
    c.table = (const int32_t*)b->table;
    c.q_start = (const int32_t*)b->q_start;
    c.kv_len = (const int32_t*)b->kv_len;
    c.status = ctx->d_status;
    c.told = ctx->d_abort + 8;
    c.heads = g->heads;
    c.kv_heads = g->kv_heads;
    c.group = g->heads / g->kv_heads;
    c.dim = g->dim;
    c.page_log2 = 0;
    while ((1u << c.page_log2) < g->page) c.page_log2++;
    c.n_pages = g->n_pages;
    c.table_ld = b->table_ld;
    c.n_seqs = b->n_seqs;
    c.rows = b->rows;
    c.shared = b->shared_len;
    return c;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

}  // namespace pg
}  // namespace runit
