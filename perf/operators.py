"""Workloads of the serving operators: page tables built from request lengths, the 8-bit KV store
with a scale per block of tokens and head, single-token attention over that cache, and token log
probabilities.  Each operator has a plain form of elementary torch operations in 32 bits (the
default) and, where `own` is true, the framework's kernels; `exact` states it in 64 bits."""
import math

import torch

own = False

D = 128                 # head_dim of every attention kernel of the framework
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -100
DEV = "cuda"


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # One decode step of 256 running sequences (256 x 1024 tokens workload): smallest call, latency.
        dict(name="tables decode 256", op="tables", seqs=256, query_min=1, query_max=1, cached_max=1087, block_size=256, pad=0),
        # All prompts of the mixed workload admitted at once: 64 prompts of 4096-8192 tokens.
        dict(name="tables prompts 64", op="tables", seqs=64, query_min=4096, query_max=8192, cached_max=2048, block_size=256, pad=0),
        # Decode step: one new token per sequence, appended to partly filled groups.
        dict(name="store decode 256", op="store", seqs=256, query_min=1, query_max=1, cached_max=1087, kv_heads=8, block_size=256, scale_block=64),
        # One chunk of a chunked prefill (budget of 8192 tokens), ragged, on top of cached prefixes.
        dict(name="store chunk 8k", op="store", seqs=11, query_min=300, query_max=1190, cached_max=2048, kv_heads=8, block_size=256, scale_block=64),
        # Whole prompts stored at once: 16 of 4096-8192 tokens, one scale per page.
        dict(name="store prompts 16", op="store", seqs=16, query_min=4096, query_max=8192, cached_max=0, kv_heads=8, block_size=256, scale_block=256),
        # 8 sequences of 16-1024 tokens, the single-operator workload of the framework's benchmark.
        dict(name="decode 8 short", op="decode", seqs=8, context_min=16, context_max=1024, q_heads=16, kv_heads=8, block_size=256, scale_block=64),
        # The headline decode batch at mid run: 256 sequences, contexts 65-1087, two query heads per KV head.
        dict(name="decode 256 mid", op="decode", seqs=256, context_min=65, context_max=1087, q_heads=16, kv_heads=8, block_size=256, scale_block=64),
        # The 8B head layout (four query heads per KV head), contexts 512-1280, one scale per 128 tokens.
        dict(name="decode 256 gqa4", op="decode", seqs=256, context_min=512, context_max=1280, q_heads=32, kv_heads=8, block_size=256, scale_block=128),
        # One long conversation: a single sequence whose tokens have to be split over the whole GPU.
        dict(name="decode 1 long", op="decode", seqs=1, context_min=131001, context_max=131001, q_heads=32, kv_heads=8, block_size=256, scale_block=64),
        # Log probability of the sampled token of one request.
        dict(name="logprobs 1", op="logprobs", rows=1, vocab=151936, dtype="bf16", top=5),
        # A decode batch that asks for alternatives.
        dict(name="logprobs 256", op="logprobs", rows=256, vocab=151936, dtype="bf16", top=20),
        # Prompt scoring: every position of a 2048-token prompt.
        dict(name="logprobs prompt 2k", op="logprobs", rows=2048, vocab=151936, dtype="bf16", top=1),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("tables", "store", "decode", "logprobs"))
    if op == "tables":
        seqs = _log(rng, 1, 512)
        most = _log(rng, 1, max(1, min(32768, 393216 // seqs)))
        return dict(op=op, seqs=seqs, query_min=rng.choice((0, 1, most)) if most > 1 else 1, query_max=most,
                    cached_max=rng.choice((0, _log(rng, 1, 8192))), block_size=rng.choice((256, 512)), pad=rng.choice((0, 0, rng.randrange(1, 300))))
    if op == "store":
        seqs = _log(rng, 1, 256)
        most = _log(rng, 1, max(1, min(16384, 98304 // seqs)))
        return dict(op=op, seqs=seqs, query_min=rng.choice((1, most)), query_max=most, cached_max=rng.choice((0, _log(rng, 1, 3000))),
                    kv_heads=rng.choice((1, 2, 4, 8)), block_size=rng.choice((256, 512)), scale_block=rng.choice((64, 128, 256)))
    if op == "decode":
        heads, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 5, 8, 16))
        seqs = _log(rng, 1, 256)
        most = _log(rng, 1, max(1, min(131072, 8 * 262144 // (seqs * heads))))
        return dict(op=op, seqs=seqs, context_min=rng.choice((1, max(1, most // 2), most)), context_max=most, q_heads=heads * group, kv_heads=heads,
                    block_size=rng.choice((256, 512)), scale_block=rng.choice((64, 128, 256)))
    vocab = _log(rng, 1000, 262144)
    return dict(op=op, rows=_log(rng, 1, max(1, min(2048, 2048 * 75000 // vocab))), vocab=vocab, dtype=rng.choice(("bf16", "fp32")), top=rng.choice((0, 1, 5, 20, 32)))


# ----------------------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n lengths over [lo, hi], evenly spaced."""
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)] if n > 1 else [hi]


def _lens(g, n, lo, hi):
    """The lengths of a batch, in an order of the seed's."""
    return torch.tensor(_spread(n, lo, hi), dtype=torch.int32, device=DEV)[torch.randperm(n, generator=g, device=DEV)]


def _tables(g, lens, block_size, width):
    """Block tables of sequences of `lens` tokens over a shuffled pool: ([B, width] int32, -1 padded; blocks of the pool)."""
    pages = (lens.long() + block_size - 1) // block_size
    blocks = lens.numel() * width + 3
    perm = torch.randperm(blocks, generator=g, device=DEV).int()
    j = torch.arange(width, device=DEV)
    at = (pages.cumsum(0) - pages)[:, None] + j
    return torch.where(j < pages[:, None], perm[at.clamp(max=blocks - 1)], -1).int(), blocks


def _pool(g, case, blocks):
    """A K or V pool in use: e4m3 rows and a power-of-two scale per block of tokens and head (keys of about unit size)."""
    bs, hk, t = case["block_size"], case["kv_heads"], case["scale_block"]
    x = torch.randn(blocks, bs, hk, D, generator=g, device=DEV)
    cache = x.mul_(96.0).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    scales = torch.exp2(torch.randint(-8, -5, (blocks, bs // t, hk), generator=g, device=DEV).float())
    return cache, scales


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    if op == "tables":
        bs, b = case["block_size"], case["seqs"]
        query, cached = _lens(g, b, case["query_min"], case["query_max"]), _lens(g, b, 0, case["cached_max"])
        width = -(-(case["query_max"] + case["cached_max"]) // bs)
        tables, blocks = _tables(g, cached, bs, width)
        free = blocks + torch.randperm(b * width, generator=g, device=DEV).int()
        return dict(case=case, query=query, cached=cached, tables=tables, free=free, tokens=int(query.sum()) + case["pad"])
    if op == "store":
        hk, b = case["kv_heads"], case["seqs"]
        query, cached = _lens(g, b, case["query_min"], case["query_max"]), _lens(g, b, 0, case["cached_max"])
        context = cached + query
        tables, blocks = _tables(g, context, case["block_size"], -(-(case["query_max"] + case["cached_max"]) // case["block_size"]))
        n = int(query.sum())
        # k and v are views of the fused projection's rows [q | k | v], two query heads per KV head.
        qkv = torch.randn(n, 4 * hk * D, generator=g, device=DEV, dtype=torch.bfloat16)
        qkv *= torch.exp(0.7 * torch.randn(n, 1, generator=g, device=DEV)).to(torch.bfloat16)
        key = qkv[:, 2 * hk * D:3 * hk * D].view(n, hk, D)
        value = qkv[:, 3 * hk * D:].view(n, hk, D)
        kc, ks = _pool(g, case, blocks)
        vc, vs = _pool(g, case, blocks)
        cu = torch.zeros(b + 1, dtype=torch.int32, device=DEV)
        cu[1:] = query.cumsum(0)
        return dict(case=case, key=key, value=value, kc=kc, ks=ks, vc=vc, vs=vs, tables=tables, context=context, cu=cu)
    if op == "decode":
        context = _lens(g, case["seqs"], case["context_min"], case["context_max"])
        tables, blocks = _tables(g, context, case["block_size"], -(-case["context_max"] // case["block_size"]))
        kc, ks = _pool(g, case, blocks)
        vc, vs = _pool(g, case, blocks)
        q = torch.randn(case["seqs"], case["q_heads"], D, generator=g, device=DEV, dtype=torch.bfloat16)
        return dict(case=case, q=q, kc=kc, ks=ks, vc=vc, vs=vs, tables=tables, context=context, workspace=None)
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.randn(rows, vocab, generator=g, device=DEV, dtype=dtype).mul_(2.5)
    token = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    peak = torch.rand(rows, generator=g, device=DEV) < 0.5  # half of the rows: a confident model, its own token asked for
    logits.scatter_(1, token[:, None], torch.where(peak, 14.0, 1.0)[:, None].to(dtype))
    return dict(case=case, logits=logits, tokens=token)


# ----------------------------------------------------------------------------- plain forms
def _plain_tables(s):
    bs, n, c, tables, free = s["case"]["block_size"], s["query"], s["cached"], s["tables"], s["free"]
    b, width = tables.shape
    have = torch.clamp((c + bs - 1) // bs, max=width)
    need = torch.where(n > 0, torch.clamp((c + n + bs - 1) // bs, max=width), have)
    want = need - have
    start = torch.cumsum(want, 0) - want
    j = torch.arange(width, device=DEV)
    at = start[:, None] + j - have[:, None]
    new = torch.where((j < need[:, None]) & (at < free.numel()), free[at.clamp(0, free.numel() - 1)], -1)
    tables.copy_(torch.where(j < have[:, None], tables, new))
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    cu_q = torch.cat((zero, torch.cumsum(n, 0).int()))
    cu_k = torch.cat((zero, torch.cumsum(c + n, 0).int()))
    i = torch.arange(s["tokens"], device=DEV)
    row = torch.searchsorted(cu_q[1:].long(), i, right=True)
    live = row < b
    row = row.clamp(max=b - 1)
    pos = torch.where(live, c[row] + i - cu_q[row], 0)
    page = tables[row, torch.clamp(pos // bs, max=width - 1)]
    slot = torch.where(live & (page >= 0), page * bs + pos % bs, -1).int()
    return dict(block_tables=tables, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, context_lens=(c + n).int(), positions=pos, slot_mapping=slot)


def _plain_scale(amax):
    """The smallest power of two s with amax / s <= 448, at least MIN_SCALE."""
    m, e = torch.frexp(amax / E4M3_MAX)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), torch.where(m > 0.5, e, e - 1)), 0).clamp(min=MIN_SCALE)


def _plain_store_one(x, cache, scales, t, groups, page, off, first):
    hk = x.shape[1]
    x = x.float()
    amax = torch.where(torch.isfinite(x), x.abs(), 0).amax(-1)
    flat = scales.view(-1, hk)
    top = torch.zeros_like(flat).index_reduce_(0, groups, amax, "amax")
    # Rows from before: those of the group that a sequence's first new token falls into.
    fpage, foff = first
    fgroup = fpage * (cache.shape[1] // t) + foff // t
    began = foff % t
    old = torch.where((began > 0)[:, None], flat[fgroup], 0)
    before = torch.zeros_like(flat)
    before[fgroup] = old
    new = torch.maximum(before, _plain_scale(top))
    rows = cache.view(-1, hk, D)
    k = torch.arange(t, device=DEV)
    at = (fgroup * t)[:, None] + k
    mine = k < began[:, None]
    ratio = (old / new[fgroup])[:, None, :, None]
    again = (rows[at].float() * torch.where(mine[:, :, None, None], ratio, 1)).to(torch.float8_e4m3fn)
    rows[at[mine]] = again[mine]
    rows[page * cache.shape[1] + off] = (x / new[groups][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    flat[groups] = new[groups]


def _plain_store(s):
    t, bs, cu, context, tables = s["case"]["scale_block"], s["case"]["block_size"], s["cu"].long(), s["context"].long(), s["tables"]
    i = torch.arange(s["key"].shape[0], device=DEV)
    seq = torch.searchsorted(cu[1:], i, right=True)
    begin = context - (cu[1:] - cu[:-1])
    pos = begin[seq] + i - cu[seq]
    page, off = tables[seq, pos // bs].long(), pos % bs
    groups = page * (bs // t) + off // t
    first = tables.gather(1, (begin // bs)[:, None]).squeeze(1).long(), begin % bs
    _plain_store_one(s["key"], s["kc"], s["ks"], t, groups, page, off, first)
    _plain_store_one(s["value"], s["vc"], s["vs"], t, groups, page, off, first)
    return dict(k_cache=s["kc"], k_scales=s["ks"], v_cache=s["vc"], v_scales=s["vs"])


def _plain_decode(s):
    case, tables, context = s["case"], s["tables"], s["context"]
    hk, t = case["kv_heads"], case["scale_block"]
    b, hq, _ = s["q"].shape
    pages = tables.clamp(min=0).long()

    def rows(cache, scales):
        x = cache[pages].float().view(b, -1, t, hk, D)
        return x.mul_(scales[pages].view(b, -1, 1, hk, 1)).view(b, -1, hk, D)

    q = s["q"].float().view(b, hk, hq // hk, D) * D ** -0.5
    score = torch.matmul(q, rows(s["kc"], s["ks"]).permute(0, 2, 3, 1))
    dead = torch.arange(score.shape[-1], device=DEV) >= context[:, None]
    score.masked_fill_(dead[:, None, None, :], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(p, rows(s["vc"], s["vs"]).transpose(1, 2)) / p.sum(-1, keepdim=True)
    return out.view(b, hq, D).to(torch.bfloat16)


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    y = x - m
    e = torch.exp(y)
    z = e.sum(-1)
    lse = m.squeeze(1) + torch.log(z)
    entropy = torch.log(z) - (e * y).sum(-1) / z
    # Unique whole-number keys, ordered as the logits are and, among equals, by the lowest index.
    bits = x.add(0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32
    key -= torch.arange(x.shape[1], device=DEV)
    ids = torch.topk(key, top, dim=-1).indices
    return dict(logprobs=x.gather(1, s["tokens"][:, None]).squeeze(1) - lse, entropies=entropy, top_tokens=ids, top_logprobs=x.gather(1, ids) - lse[:, None])


# ----------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        from hilda_vllm_b200 import kernels

        s = state
        if op == "tables":
            plan = kernels.extend_block_tables(s["tables"], s["cached"], s["query"], s["free"], s["case"]["block_size"], s["tokens"])
            return {k: plan[k] for k in ("block_tables", "cu_seqlens_q", "cu_seqlens_k", "context_lens", "positions", "slot_mapping")}
        if op == "store":
            kernels.store_kvcache_fp8_blocks(s["key"], s["value"], s["kc"], s["vc"], s["ks"], s["vs"], s["tables"], s["context"], s["cu"])
            return dict(k_cache=s["kc"], k_scales=s["ks"], v_cache=s["vc"], v_scales=s["vs"])
        if op == "decode":
            if s["workspace"] is None:  # kept by the program, as the engine keeps its decode workspace
                s["workspace"] = kernels.make_block_decode_workspace(s["case"]["seqs"], s["case"]["q_heads"], s["case"]["kv_heads"], s["q"].device)
            return kernels.paged_decode_fp8_blocks(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["tables"], s["context"], D ** -0.5, workspace=s["workspace"])
        logprobs, entropies, top_tokens, top_logprobs = kernels.token_logprobs(s["logits"], s["tokens"], s["case"]["top"])
        return dict(logprobs=logprobs, entropies=entropies, top_tokens=top_tokens, top_logprobs=top_logprobs)
    if op == "tables":
        return _plain_tables(state)
    if op == "store":
        return _plain_store(state)
    if op == "decode":
        return _plain_decode(state)
    return _plain_logprobs(state)


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    b = case["seqs"]
    if op == "decode":
        tokens = sum(_spread(b, case["context_min"], case["context_max"]))
        return {"bytes": 2 * tokens * case["kv_heads"] * (D + 4 / case["scale_block"]) + 4 * b * case["q_heads"] * D, "flops": 4 * tokens * case["q_heads"] * D}
    tokens = sum(_spread(b, case["query_min"], case["query_max"]))
    if op == "tables":
        bs = case["block_size"]
        width = -(-(case["query_max"] + case["cached_max"]) // bs)
        return {"bytes": 8 * b + 4 * tokens / bs + 4 * b * width + 12 * (tokens + case["pad"]) + 12 * b, "flops": 0}
    return {"bytes": 2 * tokens * case["kv_heads"] * (3 * D + 4 / case["scale_block"]), "flops": 4 * tokens * case["kv_heads"] * D}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    def store_one(x, cache, scales, spans):
        """By sequence and group, as the definition says it: the largest new value sets the group's power of two, which never falls while
        the group holds earlier rows; everything in it is rounded to e4m3 in units of that scale."""
        t, bs = case["scale_block"], case["block_size"]
        x, values, scales = x.double(), cache.double(), scales.double()
        for row, begin, end, pages in spans:
            at = begin
            while at < end:
                stop = min(end, at // t * t + t)
                page, off, held = pages[at // bs], at % bs, at % t
                new = x[row:row + stop - at]
                amax = new.abs().amax((0, 2))
                s = torch.exp2(torch.ceil(torch.log2(amax / E4M3_MAX)).clamp(min=-100.0))
                s = torch.where(s / 2 * E4M3_MAX >= amax, s / 2, s).clamp(min=2.0 ** -100)  # log2 may round up at a power of two
                if held:
                    was = scales[page, off // t]
                    s = torch.maximum(s, was)
                    values[page, off - held:off] = (values[page, off - held:off] * (was / s)[:, None]).to(torch.float8_e4m3fn).double()
                values[page, off:off + stop - at] = (new / s[:, None]).to(torch.float8_e4m3fn).double()
                scales[page, off // t] = s
                row += stop - at
                at = stop
        return values, scales

    s = prepare(case, seed)
    op = case["op"]
    if op == "tables":
        return None  # whole numbers only
    if op == "store":
        if case["seqs"] * (case["query_max"] / case["scale_block"] + 1) > 8000 or s["kc"].numel() > 1 << 29:
            return None
        cu, context, tables = s["cu"].tolist(), s["context"].tolist(), s["tables"].tolist()
        spans = [(cu[i], context[i] - (cu[i + 1] - cu[i]), context[i], tables[i]) for i in range(case["seqs"])]
        kv, ks = store_one(s["key"], s["kc"], s["ks"], spans)
        vv, vs = store_one(s["value"], s["vc"], s["vs"], spans)
        return dict(k_cache=kv, k_scales=ks, v_cache=vv, v_scales=vs)
    if op == "decode":
        hk, t, bs = case["kv_heads"], case["scale_block"], case["block_size"]
        group = case["q_heads"] // hk
        out = torch.zeros(case["seqs"], case["q_heads"], D, dtype=torch.float64, device=DEV)
        for i, n in enumerate(s["context"].tolist()):
            pages = s["tables"][i, :-(-n // bs)].long()
            k = s["kc"][pages].reshape(-1, hk, D)[:n].double() * s["ks"][pages].reshape(-1, hk).double().repeat_interleave(t, 0)[:n, :, None]
            v = s["vc"][pages].reshape(-1, hk, D)[:n].double() * s["vs"][pages].reshape(-1, hk).double().repeat_interleave(t, 0)[:n, :, None]
            q = s["q"][i].double().view(hk, group, D)
            w = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(D), -1)
            out[i] = torch.einsum("hgn,nhd->hgd", w, v).reshape(case["q_heads"], D)
        return out
    logprobs, entropies, tops = [], [], []
    for rows, tokens in zip(s["logits"].split(64), s["tokens"].split(64)):
        lp = torch.log_softmax(rows.double(), -1)
        logprobs.append(lp.gather(1, tokens[:, None]).squeeze(1))
        entropies.append(-(lp.exp() * lp).sum(-1))
        tops.append(lp.topk(case["top"], -1).values)
    return dict(logprobs=torch.cat(logprobs), entropies=torch.cat(entropies), top_tokens=None, top_logprobs=torch.cat(tops))
