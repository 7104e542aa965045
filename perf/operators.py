"""A serving step over a paged cache, operator by operator: what is measured, and each operator in its plain form.

Three kinds, over the model shapes that this repository's configurations name (heads / key heads / head size 14 / 2 / 64, 28 / 4 / 128 and
16 / 16 / 128, vocabularies of 50304 to 152064) and generic ones beside them:

  append     the projected rows of a batch of sequences: rotation by position, keys and values into the pages of the cache, queries out
  attention  the rows' attention over the pages: ragged lengths, one or many rows a sequence, a prefix that all sequences share, capped scores,
             a bias by distance, a window
  logprobs   log probabilities of given tokens, the entropy, the most probable alternatives

`own` False: the plain form, elementary torch operations in 32 bits (64 where 32 lose what matters), rounded once at the end.
"""
import ctypes
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MODELS = [(14, 2, 64), (28, 4, 128), (16, 16, 128), (32, 8, 128), (16, 4, 64), (8, 1, 128), (12, 12, 64)]


def _append(name, seqs, q_lo, q_hi, len_hi, model, page, proj, cache, rot):
    """Sequences that get q_lo .. q_hi new positions each, ahead of a length of at most len_hi."""
    return dict(name=name, kind="append", seqs=seqs, q_lo=q_lo, q_hi=q_hi, len_lo=q_hi, len_hi=len_hi, shared=0, heads=model[0], kv_heads=model[1], dim=model[2], page=page,
                proj=proj, cache=cache, rot=rot, lens_seed=1)


def _attention(name, seqs, q_lo, q_hi, len_lo, len_hi, model, page, cache, shared=0, cap=0.0, window=0, slopes=False):
    """Lengths between len_lo and len_hi (spread over their logarithm), the shared positions included."""
    return dict(name=name, kind="attention", seqs=seqs, q_lo=q_lo, q_hi=q_hi, len_lo=len_lo, len_hi=len_hi, shared=shared, heads=model[0], kv_heads=model[1], dim=model[2],
                page=page, cache=cache, cap=cap, window=window, slopes=slopes, lens_seed=1)


def _logprobs(name, rows, vocab, dtype, k):
    return dict(name=name, kind="logprobs", rows=rows, vocab=vocab, dtype=dtype, k=k)


def listed():
    m05, m7, olmoe = MODELS[0], MODELS[1], MODELS[2]
    return [
        # one user's decoding step: the projected row of one layer
        _append("append 1 row", 1, 1, 1, 3000, m7, 16, "f32", "f16", 128),
        # a step of a large batch
        _append("append 256 rows", 256, 1, 1, 4000, m7, 64, "bf16", "bf16", 128),
        # prompts of four users in one pass, from a projection that was kept in 32 bits
        _append("append 8000 rows", 4, 1500, 2600, 8000, olmoe, 128, "f32", "f16", 64),
        # one user's decoding step of a small model: latency
        _attention("attention 1 x 777", 1, 1, 1, 777, 777, m05, 16, "bf16"),
        # one user with a very long document
        _attention("attention 1 x 131072", 1, 1, 1, 131072, 131072, m7, 64, "f16"),
        # a decoding step of a batch of unlike lengths
        _attention("attention 64 ragged", 64, 1, 1, 60, 8100, m7, 64, "f16"),
        # a batch behind one long system prompt
        _attention("attention 128 behind 32768", 128, 1, 1, 32768 + 16, 32768 + 900, m7, 128, "bf16", shared=32768),
        # drafts of four tokens are verified by a model with windowed, distance-biased attention
        _attention("attention drafts, window", 16, 4, 4, 1500, 6000, MODELS[4], 32, "f16", window=1024, slopes=True),
        # prompts in portions behind what is cached, scores capped
        _attention("attention prompts, capped", 3, 700, 2048, 2048, 4096, olmoe, 64, "bf16", cap=30.0),
        # log probability and entropy of one sampled token
        _logprobs("logprobs 1 x 50304", 1, 50304, "f32", 0),
        # a step of eight users, each with twenty alternatives
        _logprobs("logprobs 8 x 151936", 8, 151936, "f32", 20),
        # scores of a prompt's own tokens
        _logprobs("logprobs 2048 x 152064", 2048, 152064, "bf16", 5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "logprobs"])
    if kind == "logprobs":
        vocab, dtype = _log(rng, 1000, 152064), rng.choice(["f32", "f16", "bf16"])
        c = _logprobs("", _log(rng, 1, min(8192, 155_000_000 // vocab)), vocab, dtype, rng.choice([0, 1, 5, rng.randint(2, 32)]))
        del c["name"]
        return c
    model, page, cache = rng.choice(MODELS), rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16"])
    if kind == "append":
        q_hi = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 8, 2000)])
        seqs = _log(rng, 1, min(256, 8000 // q_hi))
        c = _append("", seqs, 1, q_hi, _log(rng, q_hi, 131072), model, page, rng.choice(["f32", cache]), cache, rng.choice([0, model[2] // 2, model[2], model[2]]))
    else:
        per = model[1] * model[2]
        how = rng.choice(["step", "step", "shared", "shared", "portions"])
        cap, window, slopes = rng.choice([0.0, 0.0, 30.0, 50.0]), rng.choice([0, 0, 0, _log(rng, 64, 4096)]), rng.random() < 0.25
        if how == "step":                    # one to a few rows a sequence
            seqs, q = _log(rng, 1, 128), rng.choice([1, 1, 1, rng.randint(2, 6)])
            hi = _log(rng, 16, max(16, min(131072, 140_000_000 // (per * seqs))))
            c = _attention("", seqs, 1, q, max(q, hi // rng.randint(1, 20)), max(q, hi), model, page, cache, 0, cap, window, slopes)
        elif how == "shared":
            seqs, q = _log(rng, 2, 128), rng.choice([1, 1, 1, 2])
            pages = _log(rng, 1, max(1, min(32768, 100_000_000_000 // (seqs * q * model[0] * model[2] * 8)) // page))
            own_hi = _log(rng, 2, max(2, min(1000, 130_000_000 // (per * seqs))))
            c = _attention("", seqs, 1, q, pages * page + q, pages * page + max(q, own_hi), model, page, cache, pages * page, cap, 0, slopes)
        else:
            seqs, q = rng.randint(1, 3), _log(rng, 16, 2048)
            hi = _log(rng, q, 2 * max(q, 64))
            c = _attention("", seqs, max(1, q // 3), q, q, max(q, hi), model, page, cache, 0, cap, window, slopes)
    del c["name"]
    c["lens_seed"] = rng.randint(1, 10 ** 6)
    return c


def _lens(case):
    """Rows and lengths of the sequences."""
    rng = random.Random(case["lens_seed"])
    q = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
    own_lo, own_hi = case["len_lo"] - case["shared"], case["len_hi"] - case["shared"]
    n = [case["shared"] + max(a, _log(rng, max(1, own_lo), max(1, own_hi))) for a in q]
    return q, n


def _seen(case):
    """(pairs of a row and a key that it sees, rows of keys read): the shared positions are read once."""
    pairs = keys = 0
    for q, n in zip(*_lens(case)):
        w = case.get("window") or n
        pairs += sum(min(p + 1, w) for p in range(n - q, n))
        first = max(0, n - q + 1 - w)
        keys += n - max(first, case["shared"])
    return pairs, keys + case["shared"]


def work(case):
    if case["kind"] == "logprobs":
        size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["k"]), "flops": 5 * n}
    rows, width, kv = sum(_lens(case)[0]), case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    if case["kind"] == "append":
        size = 4 if case["proj"] == "f32" else 2
        return {"bytes": rows * (width + 2 * kv) * (size + 2), "flops": 3 * rows * (case["heads"] + case["kv_heads"]) * case["rot"]}
    pairs, keys = _seen(case)
    return {"bytes": keys * 2 * kv * 2 + 2 * rows * width * 2, "flops": 4 * pairs * width}


# ── inputs ──

def _normal(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    if case["kind"] == "logprobs":
        rows, n = case["rows"], case["vocab"]
        x = _normal(g, rows, n, std=2.5)
        # a few likely continuations in every row, some of them far ahead of the rest
        at = torch.randint(0, n, (rows, 8), generator=g, device="cuda")
        x.scatter_add_(1, at, torch.rand((rows, 8), generator=g, device="cuda") * 14)
        x[:, n - n // 64:] = -math.inf                                # ids that the tokenizer does not use
        s = dict(case=case, logits=x.to(DT[case["dtype"]]).contiguous())
        s["tokens"] = torch.where(torch.rand((rows,), generator=g, device="cuda") < 0.7, at[:, 0], torch.randint(0, n - n // 64, (rows,), generator=g, device="cuda")).int()
        s["logprob"], s["entropy"] = torch.empty((rows,), device="cuda"), torch.empty((rows,), device="cuda")
        s["top_ids"] = torch.empty((rows, case["k"]), device="cuda", dtype=torch.int32)
        s["top_logprobs"] = torch.empty((rows, case["k"]), device="cuda")
        return s
    q_lens, n_lens = _lens(case)
    seqs, page, heads, kvh, dim, shared, dt = case["seqs"], case["page"], case["heads"], case["kv_heads"], case["dim"], case["shared"], DT[case["cache"]]
    blocks = -(-max(n_lens) // page)
    used = [(n + page - 1) // page for n in n_lens]
    first = [shared // page] * seqs
    if case["kind"] == "append":             # only the pages that get rows are in this pool
        first = [(n - q) // page for q, n in zip(q_lens, n_lens)]
    total = shared // page + sum(u - f for u, f in zip(used, first))
    order = torch.randperm(total + 3, generator=g, device="cuda").cpu()
    rows = sum(q_lens)
    table = torch.zeros((seqs, blocks), dtype=torch.int32)
    at = shared // page
    for b in range(seqs):
        table[b, :shared // page] = order[:shared // page].int()
        table[b, first[b]:used[b]] = order[at:at + used[b] - first[b]].int()
        at += used[b] - first[b]
    starts = torch.zeros((seqs + 1,), dtype=torch.int32)
    starts[1:] = torch.tensor(q_lens).cumsum(0)
    s = dict(case=case, rows=rows, n_pages=total + 3, blocks=blocks, max_q=max(q_lens), max_len=max(n_lens))
    s["table"], s["q_start"], s["kv_len"] = table.cuda(), starts.cuda(), torch.tensor(n_lens, dtype=torch.int32).cuda()
    s["k_pages"], s["v_pages"] = (torch.empty((total + 3, kvh, page, dim), dtype=dt, device="cuda").normal_(0, 1, generator=g) for _ in range(2))
    if case["kind"] == "append":
        s["proj"] = _normal(g, rows, (heads + 2 * kvh) * dim).to(DT[case["proj"]])
        rot = case["rot"]
        f = torch.tensor([1e6 ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float64)
        s["freq"] = torch.stack([f.float(), (f - f.float().double()).float()]).cuda()      # the frequencies, and what their rounding has left
        s["q_out"] = torch.empty((rows, heads * dim), dtype=dt, device="cuda")
        return s
    s["q"] = _normal(g, rows, heads * dim, std=1.5).to(dt)
    s["out"] = torch.empty((rows, heads * dim), dtype=dt, device="cuda")
    s["slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)]).cuda() if case["slopes"] else None
    s["scale"] = 1 / math.sqrt(dim)
    return s


# ── the framework's operators ──

_kept = []


def _context():
    import runit_mac_b200 as R
    if not _kept:
        _kept.append(R.Context(0, stream=torch.cuda.current_stream().cuda_stream))
    return R, _kept[0]


def _call(s):
    """What a program lays down once for a layer's cache and a batch: their descriptions, and the workspace."""
    if "call" in s:
        return s["call"]
    R, ctx = _context()
    case = s["case"]
    cfg = R.PagedCfg(heads=case["heads"], kv_heads=case["kv_heads"], dim=case["dim"], page=case["page"], n_pages=s["n_pages"],
                     type=R.TYPE_F16 if case["cache"] == "f16" else R.TYPE_BF16, window=case.get("window", 0), scale=s.get("scale", 1.0), cap=case.get("cap", 0.0),
                     slopes=None if s.get("slopes") is None else s["slopes"].data_ptr(), k_pages=s["k_pages"].data_ptr(), v_pages=s["v_pages"].data_ptr())
    batch = R.PagedBatch(n_seqs=case["seqs"], rows=s["rows"], table_ld=s["blocks"], shared_len=case["shared"], table=s["table"].data_ptr(),
                         q_start=s["q_start"].data_ptr(), kv_len=s["kv_len"].data_ptr())
    n = 0 if case["kind"] == "append" else R.paged_attention_scratch_bytes(ctx, cfg, batch)
    s["scratch"] = torch.empty((max(n, 1),), dtype=torch.uint8, device="cuda")
    s["call"] = (R, ctx, ctypes.byref(cfg), ctypes.byref(batch), n)
    return s["call"]


def _run_own(s):
    case = s["case"]
    if case["kind"] == "logprobs":
        R, ctx = _context()
        kind = {"f32": R.TYPE_F32, "f16": R.TYPE_F16, "bf16": R.TYPE_BF16}[case["dtype"]]
        k = case["k"]
        R.token_logprobs(ctx, s["logits"], kind, case["vocab"], case["vocab"], case["rows"], s["tokens"], s["logprob"], s["entropy"], k,
                         s["top_ids"] if k else None, s["top_logprobs"] if k else None)
        return {n: s[n] for n in ("logprob", "entropy", "top_ids", "top_logprobs")}
    R, ctx, cfg, batch, nbytes = _call(s)
    width = case["heads"] * case["dim"]
    if case["kind"] == "append":
        kind = {"f32": R.TYPE_F32, "f16": R.TYPE_F16, "bf16": R.TYPE_BF16}[case["proj"]]
        R.paged_append(ctx, cfg, batch, s["proj"], kind, width + 2 * case["kv_heads"] * case["dim"], s["freq"] if case["rot"] else None, case["rot"], s["q_out"], width)
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    R.paged_attention(ctx, cfg, batch, s["q"], width, s["out"], width, s["scratch"], nbytes)
    return {"out": s["out"]}


# ── the plain form ──

def _plain_logprobs(s):
    x, k = s["logits"].float(), s["case"]["k"]
    n = x.shape[1]
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    logz = torch.log(z)
    mean = (e * d.clamp(min=-1e30)).sum(1, keepdim=True) / z
    logprob = torch.gather(d, 1, s["tokens"].long()[:, None]) - logz
    # values in their order, equal ones by their index
    bits = (x + 0.0).view(torch.int32)          # one zero
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 32 + (n - 1 - torch.arange(n, device=x.device))
    ids = n - 1 - (torch.topk(key, k, dim=1).values % 2 ** 32)
    return {"logprob": logprob[:, 0], "entropy": (logz - mean)[:, 0], "top_ids": ids.int(), "top_logprobs": torch.gather(d, 1, ids) - logz}


def _row_places(s):
    """Sequence and position of every row."""
    r = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["q_start"], r.int(), right=True).long() - 1
    return seq, s["kv_len"][seq].long() - s["q_start"][seq + 1].long() + r


def _plain_append(s):
    case = s["case"]
    heads, kvh, dim, rot, page = case["heads"], case["kv_heads"], case["dim"], case["rot"], case["page"]
    x = s["proj"].float().view(s["rows"], heads + 2 * kvh, dim)
    seq, pos = _row_places(s)
    angle = pos.double()[:, None] * s["freq"].double().sum(0)
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    qk = x[:, :heads + kvh]
    a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
    qk = torch.cat([a * c - b * sn, a * sn + b * c, qk[..., rot:]], -1).to(DT[case["cache"]])
    at = s["table"][seq, pos // page].long()
    s["k_pages"][at, :, pos % page] = qk[:, heads:]
    s["v_pages"][at, :, pos % page] = x[:, heads + kvh:].to(DT[case["cache"]])
    return {"q": qk[:, :heads].reshape(s["rows"], heads * dim), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attention(s):
    """Sequences side by side, padded to the longest one; the shared positions enter the products once."""
    case = s["case"]
    heads, kvh, dim, page, shared, seqs = case["heads"], case["kv_heads"], case["dim"], case["page"], case["shared"], case["seqs"]
    mq, g, first = s["max_q"], heads // kvh, shared // page
    i = torch.arange(mq, device="cuda")
    counts = (s["q_start"][1:] - s["q_start"][:-1]).long()
    rows = (s["q_start"][:-1].long()[:, None] + i).clamp(max=s["rows"] - 1)
    pos = s["kv_len"].long()[:, None] - counts[:, None] + i
    q = s["q"][rows].float().view(seqs, mq, kvh, g, dim).permute(0, 2, 3, 1, 4) * s["scale"]      # [seqs][kvh][g][mq][dim]
    own_pages = s["table"][:, first:].long()

    def pages(pool):
        return pool[own_pages].float().transpose(1, 2).reshape(seqs, kvh, -1, dim)

    def prefix(pool):
        return pool[s["table"][0, :first].long()].float().transpose(0, 1).reshape(kvh, shared, dim)

    flat = q.permute(1, 0, 2, 3, 4).reshape(kvh, seqs * g * mq, dim)
    scores = torch.matmul(q.reshape(seqs, kvh, g * mq, dim), pages(s["k_pages"]).transpose(2, 3)).view(seqs, kvh, g, mq, -1)
    if shared:
        before = torch.matmul(flat, prefix(s["k_pages"]).transpose(1, 2)).view(kvh, seqs, g, mq, shared).transpose(0, 1)
        scores = torch.cat([before, scores], -1)
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    back = pos[:, None, None, :, None] - torch.arange(scores.shape[-1], device="cuda")
    if case["slopes"]:
        scores = scores - s["slopes"].view(kvh, g, 1, 1) * back
    hidden = back < 0
    if case["window"]:
        hidden |= back >= case["window"]
    scores = scores.masked_fill_(hidden, -math.inf)
    p = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True)))
    z = p.sum(-1, keepdim=True)
    out = torch.matmul(p[..., shared:].reshape(seqs, kvh, g * mq, -1), pages(s["v_pages"])).view(seqs, kvh, g, mq, dim)
    if shared:
        more = torch.matmul(p[..., :shared].transpose(0, 1).reshape(kvh, seqs * g * mq, shared), prefix(s["v_pages"]))
        out = out + more.view(kvh, seqs, g, mq, dim).transpose(0, 1)
    out = (out / z).to(DT[case["cache"]]).permute(0, 3, 1, 2, 4).reshape(seqs, mq, heads * dim)
    return {"out": out[i < counts[:, None]]}


def run(state):
    if own:
        return _run_own(state)
    return {"logprobs": _plain_logprobs, "append": _plain_append, "attention": _plain_attention}[state["case"]["kind"]](state)


# ── the definitions in 64 bits ──

def _exact_append(s, case):
    heads, kvh, dim, half = case["heads"], case["kv_heads"], case["dim"], case["rot"] // 2
    q_lens, n_lens = _lens(case)
    pos = torch.cat([torch.arange(n - q, n, device="cuda") for q, n in zip(q_lens, n_lens)]).double()
    seq = torch.cat([torch.full((q,), b, device="cuda") for b, q in enumerate(q_lens)])
    x = s["proj"].double().view(-1, heads + 2 * kvh, dim)
    y = x.clone()
    if half:
        turn = torch.polar(torch.ones_like(pos)[:, None], pos[:, None] * (s["freq"][0].double() + s["freq"][1].double()))[:, None]
        z = torch.complex(x[..., :half], x[..., half:2 * half])[:, :heads + kvh] * turn
        y[:, :heads + kvh, :half], y[:, :heads + kvh, half:2 * half] = z.real, z.imag
    pages = s["table"][seq, (pos // case["page"]).long()].long()
    k, v = s["k_pages"].double(), s["v_pages"].double()
    k[pages, :, (pos % case["page"]).long()] = y[:, heads:heads + kvh]
    v[pages, :, (pos % case["page"]).long()] = y[:, heads + kvh:]
    return {"q": y[:, :heads].reshape(len(pos), heads * dim), "k_pages": k, "v_pages": v}


def _exact_attention(s, case):
    heads, kvh, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty((s["rows"], heads, dim), dtype=torch.float64, device="cuda")
    at = 0
    for b, (nq, n) in enumerate(zip(*_lens(case))):
        own_pages = s["table"][b, :-(-n // page)].long()
        q = s["q"][at:at + nq].double().view(nq, heads, dim)
        j, p = torch.arange(n, device="cuda"), torch.arange(n - nq, n, device="cuda")[:, None]
        seen = (j <= p) & (j > p - (case["window"] or n + 1))
        for h in range(kvh):
            k, v = (pool[own_pages, h].double().reshape(-1, dim)[:n] for pool in (s["k_pages"], s["v_pages"]))
            for head in range(h * (heads // kvh), (h + 1) * (heads // kvh)):
                t = q[:, head] @ k.T * s["scale"]
                if case["cap"]:
                    t = torch.tanh(t / case["cap"]) * case["cap"]
                if case["slopes"]:
                    t = t - s["slopes"][head].double() * (p - j)
                out[at:at + nq, head] = torch.softmax(torch.where(seen, t, -math.inf), 1) @ v
        at += nq
    return {"out": out.reshape(s["rows"], heads * dim)}


def _exact_logprobs(s, case):
    x = s["logits"].double()
    lp = torch.log_softmax(x, 1)
    p = torch.exp(lp)
    ids = torch.cat([torch.sort(part, dim=1, descending=True, stable=True).indices[:, :case["k"]].clone() for part in s["logits"].split(256)])
    return {"logprob": lp[torch.arange(len(x), device="cuda"), s["tokens"].long()], "entropy": -torch.where(p > 0, p * lp, 0.0).sum(1), "top_ids": ids.int(),
            "top_logprobs": torch.gather(lp, 1, ids)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "append": _exact_append, "attention": _exact_attention}[case["kind"]](s, case)
