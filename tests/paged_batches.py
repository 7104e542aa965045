"""Batches of sequences over a paged cache for the tests, and the operators' definitions over them in 64 bits (numpy)."""
import ctypes as C

import numpy as np

EPS = {"f16": 2.0 ** -10, "bf16": 2.0 ** -7, "f32": 2.0 ** -23}


def to_bits(x, kind):
    """f32 values as the 16-bit type's bit patterns, rounded to nearest even (NaN kept)."""
    x = np.ascontiguousarray(x, np.float32)
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, kind):
    b = np.ascontiguousarray(b, np.uint16)
    if kind == "f16":
        return b.view(np.float16).astype(np.float32)
    return (b.astype(np.uint32) << 16).view(np.float32)


def rounded(x, kind):
    return np.asarray(x, np.float32) if kind == "f32" else from_bits(to_bits(x, kind), kind)


class Batch:
    """Sequences (rows, length) over shuffled pages; whatever no row may see is `poison`."""

    def __init__(self, seed, seqs, heads, kv_heads, dim, page, kind, shared=0, extra_rows=0, poison=np.nan, spare_pages=3, table_extra=1, window=0, cap=0.0, slopes=None, scale=None):
        rng = self.rng = np.random.default_rng(seed)
        self.seqs, self.heads, self.kv_heads, self.dim, self.page, self.kind, self.shared = seqs, heads, kv_heads, dim, page, kind, shared
        self.window, self.cap, self.slopes, self.scale = window, cap, slopes, dim ** -0.5 if scale is None else scale
        first = shared // page
        self.used = [max(first, -(-n // page)) for _, n in seqs]
        self.table_ld = max(max(self.used), 1) + table_extra
        total = first + sum(u - first for u in self.used)
        self.n_pages = total + spare_pages
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(seqs), self.table_ld), -7, np.int32)          # entries behind a sequence's pages are not read
        self.table[:, :first] = order[:first]
        at = first
        for s, u in enumerate(self.used):
            self.table[s, first:u] = order[at:at + u - first]
            at += u - first
        self.q_start = np.concatenate([[0], np.cumsum([q for q, _ in seqs])]).astype(np.int32)
        self.kv_len = np.array([n for _, n in seqs], np.int32)
        self.n_rows, self.rows = int(self.q_start[-1]), int(self.q_start[-1]) + extra_rows
        shape = (self.n_pages, kv_heads, page, dim)
        self.k, self.v = (np.full(shape, poison, np.float32) for _ in range(2))
        k, v = (rounded(rng.normal(0, 1, shape), kind) for _ in range(2))
        for s, (q, n) in enumerate(seqs):
            for p in range(0, max(n, 0), page):
                pg = self.table[0 if p < shared else s, p // page]
                w = min(page, n - p)
                self.k[pg, :, :w], self.v[pg, :, :w] = k[pg, :, :w], v[pg, :, :w]
        self.q = rounded(rng.normal(0, 1.5, (self.rows, heads, dim)), kind)

    def seq_kv(self, s):
        """Keys and values [kv_heads][length][dim] of a sequence."""
        n = int(self.kv_len[s])
        pos = np.arange(n)
        pg = np.where(pos < self.shared, self.table[0, pos // self.page], self.table[s, pos // self.page])
        return (np.moveaxis(x[pg, :, pos % self.page], 1, 0).astype(np.float64) for x in (self.k, self.v))

    # ── what the calls take ──
    def upload(self, ctx, k=None, v=None):
        import runit_mac_b200 as R
        b = {"k": ctx.buffer_from(to_bits(self.k if k is None else k, self.kind)), "v": ctx.buffer_from(to_bits(self.v if v is None else v, self.kind)),
             "table": ctx.buffer_from(self.table), "q_start": ctx.buffer_from(self.q_start), "kv_len": ctx.buffer_from(self.kv_len),
             "slopes": None if self.slopes is None else ctx.buffer_from(np.asarray(self.slopes, np.float32))}
        cfg = R.PagedCfg(heads=self.heads, kv_heads=self.kv_heads, dim=self.dim, page=self.page, n_pages=self.n_pages, type=R.TYPE_F16 if self.kind == "f16" else R.TYPE_BF16,
                         window=self.window, scale=self.scale, cap=self.cap, slopes=b["slopes"].ptr if b["slopes"] else None, k_pages=b["k"].ptr, v_pages=b["v"].ptr)
        batch = R.PagedBatch(n_seqs=len(self.seqs), rows=self.rows, table_ld=self.table_ld, shared_len=self.shared, table=b["table"].ptr, q_start=b["q_start"].ptr,
                             kv_len=b["kv_len"].ptr)
        return b, cfg, batch

    def attend(self, ctx, pad=0, fill=-3.0, keep=None):
        """out [rows][heads][dim] as the kernel gives it; rows that belong to nobody hold `fill`."""
        import runit_mac_b200 as R
        b, cfg, batch = keep or self.upload(ctx)
        width = self.heads * self.dim
        ld = width + pad
        q = np.full((self.rows, ld), 99.0, np.float32)
        q[:, :width] = self.q.reshape(self.rows, width)
        qb, ob = ctx.buffer_from(to_bits(q, self.kind)), ctx.buffer_from(to_bits(np.full((self.rows, ld), fill), self.kind))
        n = R.paged_attention_scratch_bytes(ctx, cfg, batch)
        scratch = ctx.new_buffer(n)
        scratch.upload(np.full(n, 0xFF, np.uint8))                   # NaN wherever something is read that was not written
        R.paged_attention(ctx, C.byref(cfg), C.byref(batch), qb, ld, ob, ld, scratch, n)
        ctx.flush()
        out = from_bits(ob.download(np.uint16, self.rows * ld), self.kind).reshape(self.rows, ld)
        assert (out[:, width:] == rounded(fill, self.kind)).all()
        return out[:, :width].reshape(self.rows, self.heads, self.dim)

    def reference(self):
        """(out, bound on the kernel's error) [n_rows][heads][dim] in 64 bits.

        The bound: the weights are rounded to the cache's type (half a step each, eps / 2 of P.|V|; their sum is not), so is the output (eps / 2 of it).
        A score's f32 products and sums are off by at most (dim + 8) 2^-24 of scale sum |q k|, its later steps (scaling, tanh, bias, the exponent's
        argument) by a few 2^-24 of the largest magnitude that they meet, taken as 2^-20; an exponential by 2^-22.  An error d of the scores is
        one of 2 d of the normalised weights, so 2 d P.|V| of the output.  f32 sums over n keys: n 2^-24 in the worst case, of P.|V|."""
        g = self.heads // self.kv_heads
        out = np.zeros((self.n_rows, self.heads, self.dim))
        bound = np.zeros_like(out)
        for s, (nq, n) in enumerate(self.seqs):
            k, v = self.seq_kv(s)
            for i in range(nq):
                r, p = int(self.q_start[s]) + i, n - nq + i
                if p < 0:
                    continue
                lo = max(0, p + 1 - self.window) if self.window else 0
                for h in range(self.heads):
                    kk, vv = k[h // g, lo:p + 1], v[h // g, lo:p + 1]
                    x = self.q[r, h].astype(np.float64)
                    t = kk @ x * self.scale
                    d = (self.dim + 8) * 2.0 ** -24 * np.max(np.abs(kk) @ np.abs(x)) * abs(self.scale)
                    top = np.max(np.abs(t))
                    if self.cap:
                        t = self.cap * np.tanh(t / self.cap)
                    if self.slopes is not None:
                        bias = float(np.float32(self.slopes[h])) * (p - np.arange(lo, p + 1))
                        t = t - bias
                        top = max(top, np.max(np.abs(bias)))
                    w = np.exp(t - t.max())
                    w /= w.sum()
                    with np.errstate(invalid="ignore"):
                        out[r, h] = w @ vv
                        pv = w @ np.abs(vv)
                    half = EPS[self.kind] / 2
                    bound[r, h] = half * np.abs(out[r, h]) + (half + 2 * (d + top * 2.0 ** -20 + 2.0 ** -21) + len(w) * 2.0 ** -24) * pv * (1 + half)
        return out, bound


def check(batch, got, what=""):
    ref, bound = batch.reference()
    got = got[:batch.n_rows].astype(np.float64)
    assert np.isfinite(got).all(), "%s: not finite at %s" % (what, np.argwhere(~np.isfinite(got))[:4])
    off = np.abs(got - ref) - bound
    tiny = 2.0 ** -25 if batch.kind == "f16" else 0.0                 # below f16's normal range a step is 2^-24
    assert (off <= tiny).all(), "%s: %d of %d beyond the bound, worst %.3g (value %.4g) at %s" % (
        what, (off > tiny).sum(), off.size, off.max(), ref.flat[off.argmax()], np.unravel_index(off.argmax(), off.shape))
