"""Cases of the 8-bit paged KV cache (append with rotation, decode, prefill) and of token sampling.

The cache holds e4m3 numbers, (layers, blocks, block size, KV heads, head dim), and one power-of-two
scale for each (layer, block, KV head) of keys and of values: an entry stands for code * scale.

``own`` false: the plain form, elementary torch operations in 32 bits (64 for angles of far positions
and for the sums that a sampled token is decided by).  ``own`` true: the package's calls."""
import math

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ROPE_THETA = 500000.0
LAYERS, LAYER = 2, 1     # every cache has two layers and the calls work on the second


# ---- cases ----------------------------------------------------------------------------------
def _append(name, chunks, chunk_lo, chunk_hi, prior_hi, decodes, ctx_hi, hq, hkv, dim, block, dtype, pattern):
    return dict(name=name, op="append", chunks=chunks, chunk_lo=chunk_lo, chunk_hi=chunk_hi,
                prior_hi=prior_hi, decodes=decodes, ctx_hi=ctx_hi, hq=hq, hkv=hkv, dim=dim,
                block=block, dtype=dtype, pattern=pattern)


def _decode(name, seqs, lens, ctx_lo, ctx_hi, hq, hkv, dim, block, dtype, pattern):
    return dict(name=name, op="decode", seqs=seqs, lens=lens, ctx_lo=ctx_lo, ctx_hi=ctx_hi, hq=hq,
                hkv=hkv, dim=dim, block=block, dtype=dtype, pattern=pattern)


def _prefill(name, chunks, chunk_lo, chunk_hi, prior_hi, decodes, ctx_hi, hq, hkv, dim, block, dtype, pattern):
    c = _append(name, chunks, chunk_lo, chunk_hi, prior_hi, decodes, ctx_hi, hq, hkv, dim, block, dtype, pattern)
    c["op"] = "prefill"
    return c


def _sample(name, rows, vocab, dtype, params, pattern):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, dtype=dtype, params=params, pattern=pattern)


def listed():
    return [
        # the new tokens of a small decode step (8 sequences, 12/12 heads of 64)
        _append("append-step-8", 0, 0, 0, 0, 8, 512, 12, 12, 64, 16, "f16", 1),
        # the new tokens of a full decode step: 256 sequences, 32/8 heads of 128
        _append("append-step-256", 0, 0, 0, 0, 256, 4096, 32, 8, 128, 16, "bf16", 2),
        # a mixed step: 16 prompt chunks on top of cached prefixes, packed with 240 decodes
        _append("append-mixed", 16, 128, 2048, 2048, 240, 4096, 32, 8, 128, 16, "bf16", 3),
        # the smallest decode batch: latency counts; 32-bit queries
        _decode("decode-8-f32", 8, "uniform", 1, 512, 12, 12, 64, 16, "f32", 4),
        # decode at scale: 256 sequences, lognormal contexts
        _decode("decode-256", 256, "lognormal", 16, 4096, 32, 8, 128, 16, "bf16", 5),
        # few sequences with long contexts, as a long-context server holds them
        _decode("decode-long", 14, "uniform", 8192, 32768, 32, 8, 128, 16, "bf16", 6),
        # a handful of short prompts entering an idle server
        _prefill("prefill-short", 5, 1, 200, 0, 0, 0, 32, 8, 64, 16, "f16", 7),
        # the attention of the mixed step
        _prefill("prefill-mixed", 16, 128, 2048, 2048, 240, 4096, 32, 8, 128, 16, "bf16", 8),
        # one long prompt
        _prefill("prefill-8k", 1, 8192, 8192, 0, 0, 0, 32, 8, 128, 16, "bf16", 9),
        # one user's next token
        _sample("sample-1", 1, 32000, "bf16", "mixed", 10),
        # a full batch, every row with its own parameters
        _sample("sample-256-mixed", 256, 128256, "f32", "mixed", 11),
        # a full batch drawn from the whole distribution
        _sample("sample-256-free", 256, 128256, "bf16", "free", 12),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill", "sample"])
    pattern = rng.randrange(1 << 20)
    heads = rng.choice([(12, 12, 64), (32, 8, 128), (32, 8, 64), (16, 2, 128)])
    two = rng.choice(["bf16", "f16"])
    if op == "append":
        chunks, decodes = rng.choice([(0, _spread(rng, 1, 256)), (_spread(rng, 1, 16), rng.randrange(0, 200))])
        c = _append("", chunks, 1, _spread(rng, 2, 1900), rng.randrange(0, 2000), decodes, 4096,
                    *heads, rng.choice([8, 16, 32]), rng.choice(["bf16", "f16", "f32"]), pattern)
    elif op == "decode":
        hi = _spread(rng, 20, 32768)
        seqs = max(1, min(_spread(rng, 1, 256), 400000 // hi))
        c = _decode("", seqs, rng.choice(["uniform", "lognormal"]), 1, hi,
                    *rng.choice([heads, (28, 4, 128), (40, 8, 128), (6, 2, 64)]),
                    rng.choice([8, 16, 32]), rng.choice(["bf16", "f16", "f32"]), pattern)
    elif op == "prefill":
        c = _prefill("", _spread(rng, 1, 12), 1, _spread(rng, 8, 2000), rng.randrange(0, 2000),
                     rng.choice([0, rng.randrange(0, 200)]), 4096, *heads, rng.choice([16, 32]), two, pattern)
    else:
        c = _sample("", _spread(rng, 1, 256), _spread(rng, 100, 128256), rng.choice(["bf16", "f16", "f32"]),
                    rng.choice(["mixed", "free", "top_p", "top_k"]), pattern)
    del c["name"]
    return c


# ---- structure: lengths and blocks, from the case alone ---------------------------------------
def _context_lens(case):
    rng = np.random.default_rng(case["pattern"])
    if case["lens"] == "uniform":
        return rng.integers(case["ctx_lo"], case["ctx_hi"] + 1, size=case["seqs"])
    x = np.exp(rng.normal(math.log(max(1.0, case["ctx_hi"] / 4)), 0.8, size=case["seqs"]))
    return np.clip(np.rint(x), case["ctx_lo"], case["ctx_hi"]).astype(np.int64)


def _step_lens(case):
    """(tokens cached before, new tokens) of each sequence: prompt chunks, then decodes."""
    rng = np.random.default_rng(case["pattern"])
    new = rng.integers(case["chunk_lo"], case["chunk_hi"] + 1, size=case["chunks"])
    prior = rng.integers(0, case["prior_hi"] + 1, size=case["chunks"])
    dec = np.exp(rng.normal(math.log(max(1.0, case["ctx_hi"] / 4)), 0.8, size=case["decodes"]))
    dec = np.clip(np.rint(dec), 1, max(1, case["ctx_hi"])).astype(np.int64)
    return (np.concatenate([prior, dec - 1]).astype(np.int64),
            np.concatenate([new, np.ones(case["decodes"], np.int64)]).astype(np.int64))


def _blocks(pattern, ctx, block):
    """Block tables (-1 padded) handed out from a shuffled pool with a twentieth to spare."""
    need = -(-ctx // block)
    total = int(math.ceil(need.sum() * 1.05)) + 1
    order = np.random.default_rng(pattern + 1).permutation(total).astype(np.int32)
    table = np.full((len(ctx), max(1, int(need.max()))), -1, np.int32)
    ends = np.cumsum(need)
    for i, (n, e) in enumerate(zip(need, ends)):
        table[i, :n] = order[e - n:e]
    return table, total


# ---- the 8-bit form -----------------------------------------------------------------------------
def _scale_for(amax):
    """The smallest power of two s with amax <= 448 s (2^-100 at least)."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e.int() - 9 + (m > 0.875).int(), -100).clamp_min(-100)
    return ((e + 127) << 23).view(torch.float32)


def _store(x, scale):
    """x / scale as e4m3 numbers; what is not finite is held as NaN."""
    return torch.where(x.isfinite(), x / scale, math.nan).to(torch.float8_e4m3fn)


def _cache(g, total, block, heads, dim):
    """A filled layer pair: values whose size varies by head and channel, held in 8 bits."""
    shape = (LAYERS, total, block, heads, dim)
    x = torch.empty(shape, device="cuda").normal_(generator=g)
    x *= torch.empty((heads, dim), device="cuda").normal_(generator=g).mul_(0.5).exp_()
    s = _scale_for(x.abs().amax(dim=(2, 4)))
    return _store(x, s[:, :, None, :, None]), s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = dict(op=case["op"], dtype=dt)

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def normal(*shape):
        return torch.empty(shape, device="cuda").normal_(generator=g)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = normal(rows, vocab) * 2.5
        hot = torch.randint(0, vocab, (rows, 8), device="cuda", generator=g)
        x.scatter_add_(1, hot, normal(rows, 8).abs() * 6)  # a few likely tokens a row
        st["logits"] = x.to(dt)
        st["uniform"] = torch.rand(rows, device="cuda", generator=g)
        t = torch.empty(rows, device="cuda").uniform_(0.6, 1.3, generator=g)
        k = torch.randint(1, 200, (rows,), device="cuda", generator=g, dtype=torch.int32)
        p = torch.empty(rows, device="cuda").uniform_(0.5, 1.0, generator=g)
        m = torch.empty(rows, device="cuda").uniform_(0.0, 0.1, generator=g)
        lane = torch.arange(rows, device="cuda") % 5
        mode = case["params"]
        if mode == "mixed":  # greedy, top-k, top-p, both, min-p: as users of one server differ
            t = torch.where(lane == 4, 0.0, t)
            k = torch.where((lane == 0) | (lane == 2), k, 0)
            p = torch.where((lane == 0) | (lane == 1), p, 1.0)
            m = torch.where(lane == 3, m, 0.0)
        else:
            k = k if mode == "top_k" else torch.zeros_like(k)
            p = p if mode == "top_p" else torch.ones_like(p)
            m = torch.zeros_like(m)
        st.update(temperature=t, top_k=k.int(), top_p=p, min_p=m)
        return st

    hq, hkv, dim, block = case["hq"], case["hkv"], case["dim"], case["block"]
    if case["op"] == "decode":
        ctx = _context_lens(case)
        prior, new = ctx - 1, np.ones_like(ctx)
    else:
        prior, new = _step_lens(case)
        ctx = prior + new
    table, total = _blocks(case["pattern"], ctx, block)
    st["key_cache"], st["key_scale"] = _cache(g, total, block, hkv, dim)
    st["value_cache"], st["value_scale"] = _cache(g, total, block, hkv, dim)
    st["max_ctx"], st["max_new"] = int(ctx.max()), int(new.max())
    cu = np.concatenate([[0], np.cumsum(new)])
    if case["op"] == "append":
        seq = np.repeat(np.arange(len(new)), new)
        pos = np.arange(cu[-1]) - cu[seq] + prior[seq]
        slots = table[seq, pos // block].astype(np.int64) * block + pos % block
        # the slots of the touched blocks that hold tokens now
        first = prior // block * block
        upto = np.concatenate([[0], np.cumsum(ctx - first)])
        own_seq = np.repeat(np.arange(len(new)), ctx - first)
        held = np.arange(upto[-1]) - upto[own_seq] + first[own_seq]
        # rows of a captured step that stand for no sequence have slot -1
        pad = 3
        st["qkv"] = (normal(len(slots) + pad, (hq + 2 * hkv) * dim) * 1.5).to(dt)
        st["positions"] = dev(np.concatenate([pos, np.zeros(pad, np.int64)]))
        st["slots"] = dev(np.concatenate([slots, np.full(pad, -1, np.int64)]))
        st["read_slots"] = dev(table[own_seq, held // block].astype(np.int64) * block + held % block)
        st["inv_freq"] = 1.0 / (ROPE_THETA ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float32) / dim))
        st["hq"] = hq
        return st
    st["query"] = (normal(int(cu[-1]), hq, dim) * 1.5).to(dt)
    st["block_tables"], st["context_lens"] = dev(table), dev(ctx.astype(np.int32))
    st["cu_seqlens"] = dev(cu.astype(np.int64))
    st["scale"] = 1.0 / math.sqrt(dim)
    # what the program that made the batch knows on the host
    st["chunks"] = [(i, int(cu[i]), int(cu[i + 1]), int(ctx[i])) for i in range(len(new)) if new[i] > 1]
    st["chunk_blocks"] = int(sum(-(-ctx[i] // block) for i in range(len(new)) if new[i] > 1))
    st["single"] = dev(np.flatnonzero(new == 1))
    return st


# ---- plain forms --------------------------------------------------------------------------------
def _values(cache, scale, blocks):
    return cache[LAYER][blocks].float() * scale[LAYER][blocks][..., None, :, None]


def _plain_append_one(x, cache, scale, slots):
    block = cache.shape[2]
    blk, off = slots // block, slots % block
    uniq, at = torch.unique(blk, return_inverse=True)
    finite = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)                     # (rows, heads)
    index = at[:, None].expand_as(finite)
    amax = torch.zeros((uniq.numel(), x.shape[1]), device=x.device).scatter_reduce(0, index, finite, "amax")
    fresh = torch.zeros(uniq.numel(), device=x.device).scatter_reduce(0, at, (off == 0).float(), "amax") > 0
    old = scale[LAYER][uniq]
    new = torch.where(fresh[:, None], _scale_for(amax), torch.maximum(old, _scale_for(amax)))
    grown = (new != old) & ~fresh[:, None]
    held = cache[LAYER][uniq]
    again = (held.float() * (old / new)[:, None, :, None]).to(torch.float8_e4m3fn)
    codes = torch.where(grown[:, None, :, None], again.float(), held.float())
    codes[at, off] = _store(x, new[at][..., None]).float()
    cache.view(torch.uint8)[LAYER, uniq] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
    scale[LAYER, uniq] = new


def _rotated(x, positions, inv_freq):
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _plain_append(st):
    heads, dim = st["key_cache"].shape[3:]
    n, hq = st["qkv"].shape[0], st["hq"]
    q, k, v = st["qkv"].view(n, -1, dim).split([hq, heads, heads], dim=1)
    keep = st["slots"] >= 0
    _plain_append_one(_rotated(k, st["positions"], st["inv_freq"])[keep], st["key_cache"], st["key_scale"], st["slots"][keep])
    _plain_append_one(v.float()[keep], st["value_cache"], st["value_scale"], st["slots"][keep])
    blk = st["read_slots"] // st["key_cache"].shape[2]
    off = st["read_slots"] % st["key_cache"].shape[2]
    kv = [(c[LAYER][blk, off].float() * s[LAYER][blk][..., None]).to(torch.bfloat16)
          for c, s in ((st["key_cache"], st["key_scale"]), (st["value_cache"], st["value_scale"]))]
    return _rotated(q, st["positions"], st["inv_freq"]).to(st["dtype"]), kv[0], kv[1]


def _plain_attend(q, k, v, scale, seen):
    """q (..., rows, hq, dim), k and v (..., context, hkv, dim), seen (..., rows, context)."""
    g = q.shape[-2] // k.shape[-2]
    q = q.float().unflatten(-2, (k.shape[-2], g)).movedim(-4, -2).flatten(-3, -2)  # (..., hkv, g*rows, dim)
    s = q @ k.transpose(-3, -2).transpose(-2, -1)
    s = (s * scale).unflatten(-2, (g, -1)).masked_fill(~seen[..., None, None, :, :], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    o = (p / p.sum(-1, keepdim=True)).flatten(-3, -2) @ v.transpose(-3, -2)
    return o.unflatten(-2, (g, -1)).movedim(-2, -4).flatten(-3, -2)


def _plain_decode(st, rows):
    table = st["block_tables"][rows].long().clamp_min(0)
    k = _values(st["key_cache"], st["key_scale"], table).flatten(1, 2)
    v = _values(st["value_cache"], st["value_scale"], table).flatten(1, 2)
    seen = torch.arange(k.shape[1], device=k.device) < st["context_lens"][rows][:, None]
    return _plain_attend(st["query"][st["cu_seqlens"][rows]][:, None], k, v, st["scale"], seen[:, None])[:, 0]


def _plain_prefill(st):
    out = torch.empty_like(st["query"])
    for i, lo, hi, ctx in st["chunks"]:  # every prompt chunk has sizes of its own
        table = st["block_tables"][i, :-(-ctx // st["key_cache"].shape[2])].long()
        k = _values(st["key_cache"], st["key_scale"], table).flatten(0, 1)[:ctx]
        v = _values(st["value_cache"], st["value_scale"], table).flatten(0, 1)[:ctx]
        pos = torch.arange(ctx - (hi - lo), ctx, device=k.device)
        seen = torch.arange(ctx, device=k.device) <= pos[:, None]
        out[lo:hi] = _plain_attend(st["query"][lo:hi], k, v, st["scale"], seen).to(out.dtype)
    if st["single"].numel():
        out[st["cu_seqlens"][st["single"]]] = _plain_decode(st, st["single"]).to(out.dtype)
    return out


def _plain_sample(st):
    x = st["logits"].double()
    t = st["temperature"].double()[:, None]
    x = x / torch.where(t > 0, t, 1.0)
    y, order = x.sort(dim=-1, descending=True, stable=True)  # ties: the lowest index first
    rank = torch.arange(x.shape[1], device=x.device)
    k = st["top_k"][:, None]
    every = (y - y[:, :1]).exp()
    w = torch.where((rank < k) | (k <= 0), every, 0.0)
    before = w.cumsum(-1) - w
    p = st["top_p"].double()[:, None]
    kept = (before < p * w.sum(-1, keepdim=True)) | (p >= 1) | (rank == 0)
    w = torch.where(kept & (w >= st["min_p"].double()[:, None]) & (w > 0), w, 0.0)
    w = torch.where((t > 0) | (rank == 0), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    cum = w.cumsum(-1)
    hit = (cum > st["uniform"].double()[:, None] * cum[:, -1:]) & (w > 0)
    token = torch.where(hit, rank, x.shape[1]).amin(-1)
    chosen = x.gather(1, token[:, None])[:, 0] - y[:, 0]
    return token, (chosen - every.sum(-1).log()).float()


# ---- one pass -------------------------------------------------------------------------------------
_modules = []


def _package():
    if not _modules:
        import __graft_entry__
        __graft_entry__.load_package()
        from llm_serving_b200 import paged_ops, sampling
        _modules.extend((paged_ops, sampling))
    return _modules


def _own(st):
    ops, sampling = _package()
    if st["op"] == "sample":
        return sampling.sample(st["logits"], st["uniform"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])
    cache = (st["key_cache"], st["value_cache"], st["key_scale"], st["value_scale"], LAYER)
    if st["op"] == "append":
        q = ops.rope_reshape_and_cache_fp8(st["qkv"], st["positions"], st["inv_freq"], st["hq"], *cache, st["slots"])
        return (q, *ops.gather_cache_fp8(*cache, st["read_slots"], torch.bfloat16))
    if st["op"] == "decode":
        return ops.paged_decode_fp8(st["query"], *cache, st["block_tables"], st["context_lens"], st["scale"], st["max_ctx"])
    return ops.paged_prefill_fp8(st["query"], *cache, st["block_tables"], st["cu_seqlens"], st["context_lens"], st["scale"],
                                 st["max_new"], st["max_ctx"], prefill_blocks=st["chunk_blocks"])


def run(state):
    if own:
        return _own(state)
    if state["op"] == "append":
        return _plain_append(state)
    if state["op"] == "decode":
        rows = torch.arange(state["context_lens"].numel(), device=state["query"].device)
        return _plain_decode(state, rows).to(state["dtype"])
    if state["op"] == "prefill":
        return _plain_prefill(state)
    return _plain_sample(state)


# ---- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    es = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * es + case["rows"] * (5 * 4 + 8 + 4), "flops": 2 * n}
    hq, hkv, dim, block = case["hq"], case["hkv"], case["dim"], case["block"]
    if case["op"] == "decode":
        ctx = _context_lens(case)
        kv = 2 * int(ctx.sum()) * hkv * dim + 2 * int((-(-ctx // block)).sum()) * hkv * 4
        return {"bytes": kv + 2 * len(ctx) * hq * dim * es, "flops": 4 * int(ctx.sum()) * hq * dim}
    prior, new = _step_lens(case)
    ctx, n = prior + new, int(new.sum())
    if case["op"] == "append":
        held = int((ctx - prior // block * block).sum())
        rows = n * (hq + 2 * hkv) * dim * es + n * hq * dim * es + 2 * n * hkv * dim
        return {"bytes": rows + 2 * held * hkv * dim * 3, "flops": 6 * n * (hq + hkv) * dim}
    pairs = int((new * prior + new * (new + 1) // 2).sum())
    kv = 2 * int(ctx.sum()) * hkv * dim + 2 * int((-(-ctx // block)).sum()) * hkv * 4
    return {"bytes": kv + 2 * n * hq * dim * es, "flops": 4 * pairs * hq * dim}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _exact_append(st):
    n, hq = st["qkv"].shape[0], st["hq"]
    heads, dim, block = st["key_cache"].shape[3], st["key_cache"].shape[4], st["key_cache"].shape[2]
    rows = st["qkv"].double().reshape(n, hq + 2 * heads, dim)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=rows.device), st["positions"].double()[:, None] * st["inv_freq"].double())
    z = torch.complex(rows[:, :hq + heads, :dim // 2], rows[:, :hq + heads, dim // 2:]) * turn[:, None]
    rows[:, :hq + heads] = torch.cat([z.real, z.imag], -1)
    out = [rows[:, :hq]]
    slots = st["slots"].cpu().numpy()
    live = np.flatnonzero(slots >= 0)
    blocks = slots[live] // block
    for cache, scale, x in ((st["key_cache"], st["key_scale"], rows[:, hq:hq + heads]), (st["value_cache"], st["value_scale"], rows[:, hq + heads:])):
        held = cache[LAYER].double().cpu() * scale[LAYER].double().cpu()[:, None, :, None]
        size = scale[LAYER].double().cpu()
        x = x.cpu()
        for b in np.unique(blocks):
            t = torch.from_numpy(live[blocks == b])
            off = torch.from_numpy(slots[t.numpy()] % block)
            top = x[t].abs().amax(dim=(0, 2))
            need = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)))
            size[b] = need if int(off.min()) == 0 else torch.maximum(size[b], need)
            unit = size[b][None, :, None]
            if int(off.min()) > 0:
                held[b] = (held[b] / unit).float().to(torch.float8_e4m3fn).double() * unit
            held[b, off] = (x[t] / unit).float().to(torch.float8_e4m3fn).double() * unit
        out.append(held.reshape(-1, heads, dim)[st["read_slots"].cpu()].cuda())
    return tuple(out)


def _exact_attention(st):
    q = st["query"].double()
    out = torch.zeros_like(q)
    cu, ctx = st["cu_seqlens"].tolist(), st["context_lens"].tolist()
    block, heads = st["key_cache"].shape[2], st["key_cache"].shape[3]
    g = q.shape[1] // heads
    for i, c in enumerate(ctx):
        ids = st["block_tables"][i, :(c + block - 1) // block].long()
        k, v = ((cache[LAYER, ids].double() * scale[LAYER, ids].double()[:, None, :, None]).reshape(-1, heads, q.shape[2])[:c]
                for cache, scale in ((st["key_cache"], st["key_scale"]), (st["value_cache"], st["value_scale"])))
        for lo in range(cu[i], cu[i + 1], 1024):
            hi = min(lo + 1024, cu[i + 1])
            late = torch.arange(c, device=q.device)[None] > torch.arange(lo - cu[i + 1] + c, hi - cu[i + 1] + c, device=q.device)[:, None]
            for h in range(heads):
                s = torch.einsum("rgd,cd->grc", q[lo:hi, h * g:(h + 1) * g], k[:, h]) * st["scale"]
                out[lo:hi, h * g:(h + 1) * g] = torch.einsum("grc,cd->rgd", s.masked_fill(late, -math.inf).softmax(-1), v[:, h])
    return out


def _exact_sample(st):
    x = st["logits"].double().cpu().numpy()
    tokens, logs = [], []
    for r in range(x.shape[0]):
        t, k, p, m, u = (float(st[f][r]) for f in ("temperature", "top_k", "top_p", "min_p", "uniform"))
        z = x[r] / (t or 1.0)
        z = z - z.max()
        logs_all = math.log(np.exp(z).sum())
        order = np.lexsort((np.arange(len(z)), -z))
        order = order[:1] if t == 0 else order[:int(k)] if k > 0 else order
        w = np.exp(z[order])
        if p < 1:
            upto = int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")) + 1
            order, w = order[:upto], w[:upto]
        order = np.sort(order[w >= m])
        c = np.cumsum(np.exp(z[order]))
        token = int(order[min(len(order) - 1, int(np.searchsorted(c, u * c[-1], side="right")))])
        tokens.append(token)
        logs.append(z[token] - logs_all)
    return torch.tensor(tokens), torch.tensor(logs, dtype=torch.float64)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    return _exact_append(st) if case["op"] == "append" else _exact_attention(st)
