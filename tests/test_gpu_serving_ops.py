"""The serving operators on the GPU — page tables from request lengths, the block-scaled 8-bit KV
store, decode attention over that cache, token log probabilities — each against a plain statement of
its definition in 64 bits, and all of them together as one decode step.

Tolerances.  Tables, cache bytes and scales: equal.  Attention: the output's rounding to bf16
(2^-8 of it), the probabilities' rounding to 16 bits (2^-11 each, weighted by p |v|) and the fp32
score sums.  Log probabilities: fp32 sums of at most V / 1024 + 64 terms per partial sum (2^-24 of
the sum each), the exponentials (2^-21) and the rounding of their arguments (2^-23 |x - m|)."""
import math

import numpy as np
import pytest
import torch

from hilda_vllm_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128
E4M3 = torch.float8_e4m3fn


# ----------------------------------------------------------------------------- tables
def tables_ref(tables, cached, query, free, bs, max_tokens):
    tables = [list(r) for r in tables]
    width = len(tables[0]) if tables else 1
    cu_q, cu_k, ctx, pos, slot, taken, err = [0], [0], [], [], [], 0, 0
    for b, (c, n) in enumerate(zip(cached, query)):
        c, n = max(c, 0), max(n, 0)
        have = min(-(-c // bs), width)
        need = min(-(-(c + n) // bs), width) if n else have
        err |= 2 if n and c + n > width * bs else 0
        for j in range(have, width):
            tables[b][j] = -1
            if j < need:
                tables[b][j] = free[taken] if taken < len(free) else -1
                taken += 1
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + c + n)
        ctx.append(c + n)
        for p in range(c, c + n):
            page = tables[b][p // bs] if p // bs < width else -1
            pos.append(p)
            slot.append(page * bs + p % bs if page >= 0 and page * bs + p % bs < 2 ** 31 else -1)
    err |= (1 if taken > len(free) else 0) | (4 if len(pos) > max_tokens else 0)
    pos, slot = pos[:max_tokens], slot[:max_tokens]
    pos += [0] * (max_tokens - len(pos))
    slot += [-1] * (max_tokens - len(slot))
    return dict(block_tables=tables, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, context_lens=ctx, positions=pos,
                slot_mapping=slot, status=[min(taken, len(free)), err])


def check_tables(tables, cached, query, free, bs, max_tokens, device_tables=None):
    i32 = dict(dtype=torch.int32, device=DEV)
    bt = torch.tensor(tables, **i32) if device_tables is None else device_tables
    got = kernels.extend_block_tables(bt, None if cached is None else torch.tensor(cached, **i32),
                                      torch.tensor(query, **i32), torch.tensor(free, **i32), bs, max_tokens)
    want = tables_ref(tables, cached or [0] * len(query), query, free, bs, max_tokens)
    for k, v in want.items():
        assert got[k].cpu().tolist() == v, k


@pytest.mark.parametrize("b,cmax,nmax,bs,extra", [
    (1, 0, 1, 256, 0), (1, 5000, 3000, 256, 0), (7, 600, 0, 256, 0), (33, 1000, 700, 256, 5), (256, 1087, 1, 256, 0),
    (300, 70, 70, 16, 100), (1025, 40, 9, 32, 1), (4096, 700, 3, 512, 0), (64, 3000, 2000, 48, 7),
])
def test_tables_random(b, cmax, nmax, bs, extra):
    g = np.random.default_rng(b + cmax)
    cached, query = g.integers(0, cmax + 1, b).tolist(), g.integers(0, nmax + 1, b).tolist()
    cached[0], query[-1] = -3, -1  # negative lengths count as 0
    width = -(-(cmax + nmax) // bs) + 1
    tables = g.integers(0, 10000, (b, width)).tolist()
    free = (g.permutation(b * width) + 10000).tolist()
    check_tables(tables, cached, query, free, bs, sum(max(n, 0) for n in query) + extra)


@pytest.mark.parametrize("b,free,width,max_tokens", [(40, 20, 6, 4000), (40, 500, 2, 4000), (40, 500, 6, 1001), (9, 0, 6, 900),
                                                     (9, 3, 1, 0)])
def test_tables_what_does_not_fit_is_left_out_and_reported(b, free, width, max_tokens):
    g = np.random.default_rng(7)
    cached, query = g.integers(0, 300, b).tolist(), g.integers(0, 300, b).tolist()
    check_tables(g.integers(0, 99, (b, width)).tolist(), cached, query, list(range(100, 100 + free)), 100, max_tokens)


def test_tables_without_cached_lengths_in_a_wider_table_and_huge_ids():
    big = torch.full((5, 12), 77, dtype=torch.int32, device=DEV)
    query = [0, 300, 256, 257, 1]
    check_tables([[77] * 4] * 5, None, query, [9, 2 ** 31 // 256 - 1, 2 ** 31 // 256, 3, 2, 1, 8], 256, 900,
                 device_tables=big[:, 3:7])
    assert bool((big[:, :3] == 77).all()) and bool((big[:, 7:] == 77).all())


def test_tables_of_no_sequences():
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    got = kernels.extend_block_tables(none.view(0, 4), none, none, none, 256, 3)
    assert got["cu_seqlens_q"].tolist() == [0] and got["cu_seqlens_k"].tolist() == [0]
    assert got["positions"].tolist() == [0, 0, 0] and got["slot_mapping"].tolist() == [-1] * 3
    assert got["status"].tolist() == [0, 0]


def test_tables_equal_the_engines_allocator_and_prefill_metadata(seq_block_size):
    from hilda_vllm_b200.engine.block_manager import BlockManager
    from hilda_vllm_b200.engine.model_runner import prefill_metadata
    from hilda_vllm_b200.engine.scheduler import ScheduledSequence
    from hilda_vllm_b200.engine.sequence import Sequence

    seq_block_size(16)
    bm = BlockManager(200, 16)
    seqs = [Sequence(list(range(n))) for n in (5, 16, 33, 100, 1)]
    free = list(bm.free_block_ids)
    for s in seqs:
        bm.allocate_uncached(s)
    meta = prefill_metadata([ScheduledSequence(s, len(s.token_ids)) for s in seqs], 16)
    i32 = dict(dtype=torch.int32, device=DEV)
    got = kernels.extend_block_tables(torch.full((5, 7), -1, **i32), None, torch.tensor([len(s.token_ids) for s in seqs], **i32),
                                      torch.tensor(free, **i32), 16, len(meta["positions"]))
    for k in ("positions", "cu_seqlens_q", "cu_seqlens_k", "slot_mapping"):
        assert np.array_equal(got[k].cpu().numpy(), meta[k]), k
    for row, s in zip(got["block_tables"].tolist(), seqs):
        assert row == s.block_table + [-1] * (7 - len(s.block_table))


# ----------------------------------------------------------------------------- store
def scale_of(amax):
    """Smallest power of two s, at least 2^-100, with amax / s <= 448."""
    s = torch.full_like(amax, 2.0 ** -100)
    for e in range(-100, 130):
        s = torch.where(amax / s > 448, s * 2, s)
    return s


def store_ref(x, cache, scales, tables, context, cu):
    """x [N, Hk, D], cache [NB, BS, Hk, D] e4m3, scales [NB, G, Hk]; CPU; cache and scales updated."""
    nb, bs, hk, _ = cache.shape
    t = bs // scales.shape[1]
    for b, end in enumerate(context):
        n = cu[b + 1] - cu[b]
        at = end - n
        while at < end:
            stop = min(end, at // t * t + t)
            row = cu[b] + at - (end - n)
            begin, at = at, stop
            if begin < 0 or begin // bs >= len(tables[b]) or not 0 <= tables[b][begin // bs] < nb:
                continue
            page, off, held = tables[b][begin // bs], begin % bs, begin % t
            new = x[row:row + stop - begin].double()
            s = scale_of(torch.where(new.isfinite(), new.abs(), 0).amax((0, 2)))
            if held:
                old = scales[page, off // t].double()
                s = torch.maximum(s, old)
                rows = cache[page, off - held:off].double() * (old / s)[:, None]
                cache[page, off - held:off] = rows.to(E4M3)
            cache[page, off:off + stop - begin] = (new / s[:, None]).clamp(-448, 448).to(E4M3)
            scales[page, off // t] = s.float()


def same_bytes(a, b):
    a, b = a.view(torch.uint8).cpu(), b.view(torch.uint8)
    nan = ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)  # a NaN's sign is nobody's
    return bool(((a == b) | nan).all())


def pool(g, nb, bs, hk, t):
    cache = (torch.randn(nb, bs, hk, D, generator=g) * 90).clamp(-448, 448).to(E4M3)
    return cache, torch.exp2(torch.randint(-9, -4, (nb, bs // t, hk), generator=g).float())


def pages(g, lens, bs, nb, width):
    perm, rows = torch.randperm(nb, generator=g).tolist(), []
    for n in lens:
        k = -(-max(n, 0) // bs)
        rows.append([perm.pop() for _ in range(k)] + [-1] * (width - k))
    return rows


def run_store(x, y, state, tables, context, cu):
    i32 = dict(dtype=torch.int32, device=DEV)
    kernels.store_kvcache_fp8_blocks(x, y, *state, torch.tensor(tables, **i32), torch.tensor(context, **i32),
                                     None if cu is None else torch.tensor(cu, **i32))


@pytest.mark.parametrize("hk,bs,t,query,cached", [
    (8, 256, 64, [1] * 40, None), (8, 256, 64, [1, 0, 63, 64, 65, 255, 256, 257, 700], None),
    (1, 512, 256, [5, 600, 1, 0, 2000], None), (2, 256, 128, [130, 1, 1, 127], [126, 127, 128, 1]),
    (4, 768, 192, [400, 200], [191, 192]), (5, 256, 64, [3000], [0]), (3, 64, 64, [70, 1, 64], [10, 63, 64]),
    (8, 256, 256, [1] * 300, None), (32, 256, 64, [5500, 900], [0, 30]), (32, 256, 128, [9000, 2500], [0, 100]),
    # more sequences than are searched in shared memory, in all and between two rows of a window
    (1, 64, 64, [1, 0, 2] * 400, None), (2, 64, 64, [3] + [0] * 1200 + [2, 0, 50], None), (1, 64, 64, [1] * 900, None),
    (2, 128, 128, [20] * 30, None), (3, 256, 256, [40] * 20 + [250], None), (2, 256, 256, [100, 90, 120] * 5, None),
])
@pytest.mark.parametrize("explicit", [True, False])
def test_store_blocks_bit_exact(hk, bs, t, query, cached, explicit):
    if not explicit and any(q != 1 for q in query):
        pytest.skip("one row per sequence only")
    g = torch.Generator().manual_seed(hk * 1000 + t + len(query))
    cached = torch.randint(0, 2 * bs, (len(query),), generator=g).tolist() if cached is None else cached
    context = [c + q for c, q in zip(cached, query)]
    width = max(1, -(-max(context) // bs))
    nb = sum(-(-c // bs) for c in context) + 2
    tables = pages(g, context, bs, nb, width)
    cu = [0]
    for q in query:
        cu.append(cu[-1] + q)
    n = cu[-1] + (3 if explicit else 0)  # rows behind the last sequence are nobody's
    rows = torch.randn(n, 3, hk, D, generator=g) * torch.exp2(torch.randint(-6, 6, (n, 3, hk, 1), generator=g).float())
    qkv = rows.bfloat16().view(n, -1).to(DEV)
    key, value = qkv[:, hk * D:2 * hk * D].view(n, hk, D), qkv[:, 2 * hk * D:].view(n, hk, D)
    kc, ks = pool(g, nb, bs, hk, t)
    vc, vs = pool(g, nb, bs, hk, t)
    state = [x.to(DEV) for x in (kc, vc, ks, vs)]
    run_store(key, value, state, tables, context, cu if explicit else None)
    store_ref(key.cpu(), kc, ks, tables, context, cu)
    store_ref(value.cpu(), vc, vs, tables, context, cu)
    for got, want in zip(state, (kc, vc, ks, vs)):
        assert same_bytes(got, want)


def test_store_blocks_token_by_token_grows_the_scale():
    """A sequence decoded over a group's border, each token larger than the last."""
    g = torch.Generator().manual_seed(3)
    kc, ks = pool(g, 4, 256, 2, 64)
    vc, vs = pool(g, 4, 256, 2, 64)
    state = [x.to(DEV) for x in (kc, vc, ks, vs)]
    for pos in range(100):
        x = (torch.randn(1, 2, 2, D, generator=g) * 2.0 ** (pos / 6 - 9)).bfloat16()
        run_store(x[:, 0].to(DEV), x[:, 1].to(DEV), state, [[2, -1]], [pos + 1], None)
        store_ref(x[:, 0], kc, ks, [[2, -1]], [pos + 1], [0, 1])
        store_ref(x[:, 1], vc, vs, [[2, -1]], [pos + 1], [0, 1])
    for got, want in zip(state, (kc, vc, ks, vs)):
        assert same_bytes(got, want)


@pytest.mark.parametrize("hk,t,query,cached", [(2, 64, [1] * 9, None), (3, 128, [20, 1, 90, 128, 200], [5, 127, 64, 1, 0]),
                                               (2, 256, [1, 100, 400], [255, 30, 256 + 7])])
@pytest.mark.parametrize("old", [0.0, 2.0 ** -140, 2.0 ** -60, 2.0 ** 100, 0.3, 1e-39, 5e-31, 2.0 ** 127, 3e38, 7 * 2.0 ** -13])
def test_store_blocks_appends_to_groups_of_any_scale(hk, t, query, cached, old):
    """A caller's own scales, zero, no powers of two, subnormal ones and the type's largest among them: scale :=
    max(old, what the new rows need), earlier rows times old / new."""
    g = torch.Generator().manual_seed(64)
    cached = torch.randint(1, t, (len(query),), generator=g).tolist() if cached is None else cached
    context = [c + q for c, q in zip(cached, query)]
    nb = sum(-(-c // 256) for c in context) + 1
    tables, cu = pages(g, context, 256, nb, max(-(-c // 256) for c in context)), np.concatenate(([0], np.cumsum(query))).tolist()
    kc, ks = pool(g, nb, 256, hk, t)
    vc, vs = pool(g, nb, 256, hk, t)
    ks.fill_(old)
    vs.fill_(old)
    x = (torch.randn(2, cu[-1], hk, D, generator=g) * torch.exp2(torch.randint(-9, 4, (2, cu[-1], hk, 1), generator=g).float())).bfloat16()
    x[1] *= min(max(old, 1e-30), 1e30)  # values about as large as the scale, which then stays
    state = [s.to(DEV) for s in (kc, vc, ks, vs)]
    run_store(x[0].to(DEV), x[1].to(DEV), state, tables, context, cu)
    store_ref(x[0], kc, ks, tables, context, cu)
    store_ref(x[1], vc, vs, tables, context, cu)
    for got, want in zip(state, (kc, vc, ks, vs)):
        assert same_bytes(got, want)


def test_store_blocks_extreme_values():
    """Zeros, the type's smallest and largest, infinities, NaN; the borders of 448 * 2^k."""
    g = torch.Generator().manual_seed(4)
    n = 9 * 64
    x = torch.randn(n, 1, D, generator=g)
    x[:64] = 0
    x[64:128] *= 2.0 ** -130
    x[128:192] *= 2.0 ** 125
    x[192, 0, 5] = math.inf
    x[200, 0, 6] = math.nan
    x[256:320] = math.nan
    x[320:384] = -math.inf
    x[384:448] = 448.0
    x[448:512] = 450.0
    x[512:576] = 7 * 2.0 ** -108
    x = x.bfloat16()
    kc, ks = pool(g, 3, 256, 1, 64)
    vc, vs = pool(g, 3, 256, 1, 64)
    state = [t.to(DEV) for t in (kc, vc, ks, vs)]
    run_store(x.to(DEV), -x.to(DEV), state, [[2, 0, 1]], [n], [0, n])
    store_ref(x, kc, ks, [[2, 0, 1]], [n], [0, n])
    store_ref(-x, vc, vs, [[2, 0, 1]], [n], [0, n])
    for got, want in zip(state, (kc, vc, ks, vs)):
        assert same_bytes(got, want)


@pytest.mark.parametrize("hk,bs,t,query", [(8, 256, 256, [6000] * 16), (5, 256, 64, [30000, 31000, 30500]), (5, 128, 128, [40000, 41000]),
                                           (5, 64, 64, [1] * 4000)])
def test_store_blocks_large_calls_bit_exact(hk, bs, t, query):
    """As many rounds of the GPU as give a block several heads, the last block of a window fewer."""
    g = torch.Generator(device=DEV).manual_seed(hk + bs + t)
    cached = [(7 * i) % (bs - 1) for i in range(len(query))]
    context = [c + n for c, n in zip(cached, query)]
    nb, cu = sum(-(-c // bs) for c in context), np.concatenate(([0], np.cumsum(query))).tolist()
    tables = pages(torch.Generator().manual_seed(1), context, bs, nb, max(-(-c // bs) for c in context))
    x = torch.randn(2, cu[-1], hk, D, generator=g, device=DEV, dtype=torch.bfloat16)
    x *= torch.exp2(torch.randint(-6, 6, (2, cu[-1], hk, 1), generator=g, device=DEV).float()).bfloat16()
    state = [torch.randint(0, 127, (nb, bs, hk, D), generator=g, device=DEV, dtype=torch.uint8).view(E4M3) for _ in range(2)]
    state += [torch.exp2(torch.randint(-9, -4, (nb, bs // t, hk), generator=g, device=DEV).float()) for _ in range(2)]
    want = [s.cpu() for s in state]
    run_store(x[0], x[1], state, tables, context, cu)
    for i in range(2):
        store_ref(x[i].cpu(), want[i], want[2 + i], tables, context, cu)
        assert torch.equal(state[2 + i].cpu(), want[2 + i]) and same_bytes(state[i], want[i])


def test_store_blocks_skips_what_has_no_place():
    """Padding rows (context 0), pages outside the pool, positions before 0 or behind the table."""
    g = torch.Generator().manual_seed(5)
    kc, ks = pool(g, 4, 256, 2, 64)
    vc, vs = pool(g, 4, 256, 2, 64)
    state = [t.to(DEV) for t in (kc, vc, ks, vs)]
    tables = [[0, 1], [-1, -1], [4, 3], [1, 2 ** 31 - 1], [2, 2]]  # no page is written by two sequences
    context, query = [0, 5, 300, 600, 3], [1, 5, 300, 600, 7]
    cu = np.concatenate(([0], np.cumsum(query))).tolist()
    x = torch.randn(cu[-1], 2, D, generator=g).bfloat16()
    run_store(x.to(DEV), x.to(DEV), state, tables, context, cu)
    store_ref(x, kc, ks, tables, context, cu)
    store_ref(x, vc, vs, tables, context, cu)
    for got, want in zip(state, (kc, vc, ks, vs)):
        assert same_bytes(got, want)


# ----------------------------------------------------------------------------- decode
def decode_ref(q, kc, vc, ks, vs, tables, context, scale):
    """(out, per element sum_j p_j |v_j|, per head the largest sum_i |q_i k_i|), 64 bits, on the GPU."""
    b, hq, _ = q.shape
    nb, bs, hk, _ = kc.shape
    t = bs // ks.shape[1]
    out = torch.zeros(b, hq, D, dtype=torch.float64, device=DEV)
    mass, size = torch.zeros_like(out), torch.zeros(b, hq, 1, dtype=torch.float64, device=DEV)
    for i, n in enumerate(context):
        n = min(n, len(tables[i]) * bs)
        live = [j for j in range(-(-n // bs)) if 0 <= tables[i][j] < nb]
        if n <= 0 or not live:
            continue
        rows = torch.cat([torch.arange(j * bs, min(n, j * bs + bs)) for j in live])
        slot = torch.tensor(tables[i])[rows // bs] * bs + rows % bs
        slot = slot.to(DEV)
        k = kc.view(-1, hk, D)[slot].double() * ks.view(-1, hk)[slot // t].double()[:, :, None]
        v = vc.view(-1, hk, D)[slot].double() * vs.view(-1, hk)[slot // t].double()[:, :, None]
        qi = q[i].double().view(hk, hq // hk, D) * scale
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", qi, k), -1)
        out[i] = torch.einsum("hgn,nhd->hgd", p, v).reshape(hq, D)
        mass[i] = torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(hq, D)
        size[i] = torch.einsum("hgd,nhd->hgn", qi.abs(), k.abs()).amax(-1).reshape(hq, 1)
    return out, mass, size


def check_decode(q, kc, vc, ks, vs, tables, context, scale=D ** -0.5, workspace=None, errors=0, out=None):
    i32 = dict(dtype=torch.int32, device=DEV)
    ws = workspace if workspace is not None else kernels.make_block_decode_workspace(q.shape[0], q.shape[1], kc.shape[2], q.device)
    got = kernels.paged_decode_fp8_blocks(q, kc, vc, ks, vs, torch.tensor(tables, **i32), torch.tensor(context, **i32), scale,
                                          out=out, workspace=ws)
    assert kernels.decode_errors(ws) == errors
    want, mass, size = decode_ref(q, kc, vc, ks, vs, tables, context, scale)
    tol = want.abs() * 2.0 ** -8 + mass * (2.0 ** -11 + 2.0 ** -18 + 2 * 130 * 2.0 ** -23 * size) + 1e-37
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{int((~(err <= tol)).sum())} off, worst {float((err / tol).max()):.2f} of the tolerance"
    return got


def decode_case(seed, hk, group, bs, t, context, extra_width=0, spare=3):
    g = torch.Generator().manual_seed(seed)
    nb = sum(-(-max(n, 0) // bs) for n in context) + spare
    width = max(1, max(-(-n // bs) for n in context)) + extra_width
    tables = pages(g, context, bs, nb, width)
    kc, ks = pool(g, nb, bs, hk, t)
    vc, vs = pool(g, nb, bs, hk, t)
    q = torch.randn(len(context), hk * group, D, generator=g).bfloat16()
    return [x.to(DEV) for x in (q, kc, vc, ks, vs)] + [tables, context]


EDGES = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 255, 256, 257, 511, 700]


@pytest.mark.parametrize("hk,group", [(8, 2), (8, 1), (8, 4), (8, 8), (4, 2), (2, 4), (1, 8), (1, 1), (1, 16), (8, 16), (3, 3),
                                      (5, 5), (2, 7), (16, 2), (1, 9)])
def test_decode_blocks_head_layouts_and_edge_lengths(hk, group):
    check_decode(*decode_case(hk * 100 + group, hk, group, 256, 64, EDGES))


@pytest.mark.parametrize("bs,t", [(256, 128), (256, 256), (512, 64), (768, 192), (64, 64), (192, 64)])
def test_decode_blocks_page_and_scale_block_sizes(bs, t):
    check_decode(*decode_case(bs + t, 8, 2, bs, t, EDGES + [1500]))


@pytest.mark.parametrize("hk,group,context", [
    (8, 4, [70001]), (8, 2, [40000, 3, 0, 17000]), (1, 8, [100000]), (2, 2, [9000] * 5), (8, 2, [1] * 1000),
    (4, 16, [30000, 1]), (8, 1, list(range(900, 1400, 3))), (1, 2, [0, 0]), (3, 4, [20011, 20011]),
])
def test_decode_blocks_splits_over_the_gpu(hk, group, context):
    check_decode(*decode_case(len(context), hk, group, 256, 64, context))


def test_decode_blocks_ignores_what_lies_behind_the_context():
    """NaN bytes and NaN / infinite scales behind each sequence's end, in its last page too."""
    q, kc, vc, ks, vs, tables, context = decode_case(1, 4, 4, 256, 64, [1, 40, 64, 65, 200, 300])
    for cache, scales in ((kc, ks), (vc, vs)):
        keep, keep_s = torch.zeros(cache.shape[:2], dtype=torch.bool), torch.zeros(scales.shape[:2], dtype=torch.bool)
        for row, n in zip(tables, context):
            for p in range(n):
                keep[row[p // 256], p % 256] = True
                keep_s[row[p // 256], p % 256 // 64] = True
        cache.view(torch.uint8)[~keep.to(DEV)] = 0x7F
        scales[~keep_s.to(DEV)] = math.nan
    check_decode(q, kc, vc, ks, vs, tables, context)


@pytest.mark.parametrize("case", ["v_scales", "k_zero", "large_scores", "tiny_q", "huge_q", "negative_scale", "one_huge_v"])
def test_decode_blocks_ranges(case):
    q, kc, vc, ks, vs, tables, context = decode_case(11, 2, 4, 256, 64, [700, 65, 3000, 129])
    g = torch.Generator().manual_seed(12)
    scale = D ** -0.5
    if case == "v_scales":  # values that differ by 2^60 between blocks
        vs.copy_(torch.exp2(torch.randint(-40, 20, vs.shape, generator=g).float()))
    elif case == "k_zero":
        ks.zero_()
    elif case == "large_scores":
        scale = 8 * D ** -0.5
    elif case == "tiny_q":
        q.mul_(2.0 ** -100)
    elif case == "huge_q":
        q.mul_(2.0 ** 100)
        ks.mul_(2.0 ** -100)
    elif case == "negative_scale":
        scale = -(D ** -0.5)
    else:  # the token with the least weight carries the largest values
        vs[:, 1] = 2.0 ** 60
    check_decode(q, kc, vc, ks, vs, tables, context, scale)


@pytest.mark.parametrize("scales", ["half_zero", "all_zero", "tiny", "zero_at_the_largest_weight"])
def test_decode_blocks_value_scales_down_to_zero(scales):
    q, kc, vc, ks, vs, tables, context = decode_case(16, 2, 4, 256, 64, [700, 65, 30000, 129])
    if scales == "half_zero":
        vs[torch.rand(vs.shape, generator=torch.Generator().manual_seed(17)).to(DEV) < 0.5] = 0
    elif scales == "all_zero":
        vs.zero_()
    elif scales == "tiny":
        vs.fill_(2.0 ** -120)
    else:  # the first group of each sequence has the largest scores by far, and no values
        first = [row[0] for row in tables]
        ks[first, 0] = 2.0
        vs[first, 0] = 0
    check_decode(q, kc, vc, ks, vs, tables, context)


def test_decode_blocks_nan_in_a_live_row_reaches_the_output():
    q, kc, vc, ks, vs, tables, context = decode_case(13, 2, 2, 256, 64, [300, 80])
    kc.view(torch.uint8)[tables[0][1], 10, 0, 3] = 0x7F
    ws = kernels.make_block_decode_workspace(2, 4, 2, q.device)
    i32 = dict(dtype=torch.int32, device=DEV)
    got = kernels.paged_decode_fp8_blocks(q, kc, vc, ks, vs, torch.tensor(tables, **i32), torch.tensor(context, **i32), 0.1, workspace=ws)
    assert bool(got[0, :2].isnan().all()) and bool(got[0, 2:].isfinite().all()) and bool(got[1].isfinite().all())


def test_decode_blocks_pages_outside_the_pool_and_narrow_tables():
    q, kc, vc, ks, vs, tables, context = decode_case(14, 8, 2, 256, 64, [700, 300, 256, 900])
    tables[0][1], tables[1][0], tables[1][1], tables[2][0] = -1, kc.shape[0], 2 ** 31 - 1, -7
    context[3] = 100000  # behind the table's width
    check_decode(q, kc, vc, ks, vs, tables, context, errors=2)


def test_decode_blocks_page_outside_the_pool_with_nan_scales_elsewhere():
    """A missing page is left out whatever the scales of pages that nobody asked for."""
    q, kc, vc, ks, vs, tables, context = decode_case(15, 2, 4, 256, 64, [700, 300])
    spare = (set(range(kc.shape[0])) - {p for row in tables for p in row}).pop()
    for x in (kc, vc, ks, vs):
        x.view(torch.uint8)[[0, spare]] = x.view(torch.uint8)[[spare, 0]]
    tables = [[{0: spare, spare: 0}.get(p, p) for p in row] for row in tables]
    assert all(0 not in row for row in tables)  # page 0 of the pool is the one that nobody asks for
    ks[0] = vs[0] = math.nan
    tables[0][1] = tables[1][0] = -1
    check_decode(q, kc, vc, ks, vs, tables, context, errors=2)


def test_decode_blocks_workspace_serves_calls_of_every_size_and_strided_rows():
    ws = kernels.make_block_decode_workspace(256, 32, 8, torch.device(DEV))
    for seed, (hk, group, context) in enumerate([(8, 4, [5000, 1, 77]), (8, 1, [400] * 200), (8, 3, [30000]), (8, 4, [64])]):
        q, kc, vc, ks, vs, tables, context = decode_case(seed, hk, group, 256, 64, context, extra_width=seed)
        wide = torch.zeros(len(context), hk * group + 6, D, dtype=torch.bfloat16, device=DEV)
        wide[:, 2:-4] = q
        out = torch.zeros(len(context), hk * group + 2, D, dtype=torch.bfloat16, device=DEV)
        check_decode(wide[:, 2:-4], kc, vc, ks, vs, tables, context, workspace=ws, out=out[:, 1:-1])
        assert not out[:, 0].any() and not out[:, -1].any()


def test_decode_blocks_4096_sequences():
    """The largest batch: short, partly empty contexts that share a few pages."""
    q, kc, vc, ks, vs, tables, _ = decode_case(72, 2, 4, 256, 64, [500] * 8)
    g = torch.Generator().manual_seed(73)
    context = torch.randint(0, 400, (4096,), generator=g).tolist()
    context[::5] = [0] * len(context[::5])
    q = torch.randn(4096, 8, D, generator=g).bfloat16().to(DEV)
    check_decode(q, kc, vc, ks, vs, [tables[i % 8] for i in range(4096)], context)


def test_decode_blocks_repeats_bit_for_bit():
    q, kc, vc, ks, vs, tables, context = decode_case(21, 8, 4, 256, 64, [30000, 5, 900, 12000])
    first = check_decode(q, kc, vc, ks, vs, tables, context)
    ws = kernels.make_block_decode_workspace(4, 32, 8, q.device)
    for _ in range(10):
        assert torch.equal(first, check_decode(q, kc, vc, ks, vs, tables, context, workspace=ws))


@pytest.mark.parametrize("share", [0.999, 0.9999])
@pytest.mark.parametrize("context,seqs", [(1000, 300), (8192, 296), (32768, 256)])
@pytest.mark.parametrize("sink", ["zero", "small"])
def test_decode_blocks_with_a_token_that_takes_nearly_all_the_weight(sink, context, seqs, share):
    """Token 0 has `share` of the weight and values of (nearly) nothing, so that the small weights of the
    others make up the output; as many sequences as let one warp walk most of one.  All of them read the
    same pages, and half of the heads have values of one sign."""
    hk, bs, t, scale = 8, 256, 64, D ** -0.5
    g = torch.Generator(device=DEV).manual_seed(71)
    nb = -(-context // bs)
    kc = (torch.randn(nb, bs, hk, D, generator=g, device=DEV) * 90).clamp(-448, 448)
    vc = (torch.randn(nb, bs, hk, D, generator=g, device=DEV) * 90).clamp(-448, 448)
    vc[:, :, ::2] = vc[:, :, ::2].abs()
    kc[..., 0] = 0
    kc[0, 0] = 0
    kc[0, 0, :, 0] = 256
    vc[0, 0] = 0 if sink == "zero" else 2.0 ** -9
    kc, vc = kc.to(E4M3), vc.to(E4M3)
    ks = torch.exp2(torch.randint(-8, -5, (nb, bs // t, hk), generator=g, device=DEV).float())
    vs = torch.exp2(torch.randint(-8, -5, (nb, bs // t, hk), generator=g, device=DEV).float())
    q = torch.randn(seqs, hk, D, generator=g, device=DEV).bfloat16()
    k = (kc.float() * ks.repeat_interleave(t, 1)[..., None]).view(-1, hk, D)[1:context]
    others = torch.logsumexp(torch.einsum("bhd,nhd->bhn", q.float(), k) * scale, -1)
    q[:, :, 0] = ((others + math.log(share / (1 - share))) / (scale * 256 * ks[0, 0])).bfloat16()
    check_decode(q, kc, vc, ks, vs, [list(range(nb))] * seqs, [context] * seqs)


def test_store_and_decode_blocks_behind_4_gib_of_cache():
    nb, bs, hk, t = 17000, 256, 8, 64  # 4.5 GB of keys, as much of values
    cache = torch.zeros(2, nb, bs, hk, D, dtype=torch.uint8, device=DEV).view(E4M3)
    scales = torch.ones(2, nb, bs // t, hk, device=DEV)
    g = torch.Generator().manual_seed(6)
    x = torch.randn(2, 300, hk, D, generator=g).bfloat16().to(DEV)
    tables, context = [[nb - 1, nb - 2]], [300]
    run_store(x[0], x[1], [cache[0], cache[1], scales[0], scales[1]], tables, context, [0, 300])
    q = torch.randn(1, 16, D, generator=g).bfloat16().to(DEV)
    check_decode(q, cache[0], cache[1], scales[0], scales[1], tables, context)
    back = cache[:, nb - 1].float() * scales[:, nb - 1].repeat_interleave(t, 1)[..., None]
    assert bool(((back - x[:, :256].float()).abs() <= 2.0 ** -4 * x[:, :256].float().abs() + 2.0 ** -9 * scales[:, nb - 1].amax()).all())
    assert not cache.view(torch.uint8)[:, :nb - 2].any()


# ----------------------------------------------------------------------------- log probabilities
def check_logprobs(x, tokens, top):
    """x [R, V] on the GPU, finite or -inf, with a finite logit in every row."""
    lp, ent, ids, tlp = kernels.token_logprobs(x, tokens, top)
    rows, vocab = x.shape
    d = x.double()
    m = d.amax(-1, keepdim=True)
    y = torch.where(d == -math.inf, 0, d - m)
    e = torch.where(d == -math.inf, 0, torch.exp(d - m))
    z = e.sum(-1, keepdim=True)
    ln_z = torch.log(z)
    spread = (e * y.abs()).sum(-1, keepdim=True) / z
    terms = vocab / 1024 + 64
    d_ln_z = terms * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -23 * spread
    want = d - m - ln_z
    tol = d_ln_z + 2.0 ** -23 * ((d - m).abs() + ln_z.abs() + 1)
    inside = (tokens >= 0) & (tokens < vocab)
    at = tokens.clamp(0, vocab - 1)[:, None]
    picked = torch.where(inside[:, None], want.gather(1, at), -math.inf).squeeze(1)
    close(lp, picked, tol.gather(1, at).squeeze(1))
    h = (ln_z + (e * y.abs()).sum(-1, keepdim=True) / z).squeeze(1)
    second = (e * y * y).sum(-1, keepdim=True) / z
    close(ent, h, (d_ln_z * (1 + spread) + 2.0 ** -22 * (1 + second + spread + ln_z)).squeeze(1))
    order = torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ids, order)
    close(tlp, want.gather(1, order), tol.gather(1, order))


def close(got, want, tol):
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    assert bool((same | ((got - want).abs() <= tol)).all()), f"worst {float(((got - want).abs() / tol)[~same].max()):.2f} of the tolerance"


@pytest.mark.parametrize("rows,vocab,top", [(1, 151936, 20), (3, 151936, 32), (300, 50257, 5), (700, 1000, 1), (2, 1, 1), (5, 2, 2),
                                            (4, 31, 31), (4, 33, 32), (7, 8191, 0), (16, 262144, 20), (40, 4097, 20), (2, 1025, 32),
                                            (2048, 300, 3), (150, 32003, 32), (1, 3000017, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_random(rows, vocab, top, dtype):
    g = torch.Generator(device=DEV).manual_seed(vocab + rows)
    x = (torch.randn(rows, vocab, generator=g, device=DEV) * 3).to(dtype)
    check_logprobs(x, torch.randint(0, vocab, (rows,), generator=g, device=DEV), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", ["equal", "few_values", "masked", "one_left", "last", "spread", "zeros", "ascending", "huge_first",
                                  "outside"])
def test_logprobs_ties_masks_and_ranges(case, dtype):
    g = torch.Generator(device=DEV).manual_seed(9)
    rows, vocab, top = 6, 20011, 32
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 3
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    if case == "equal":
        x.fill_(-2.5)
    elif case == "few_values":
        x = torch.randint(0, 3, x.shape, generator=g, device=DEV).float()
    elif case == "masked":  # all but a handful are masked, and the asked token is not or is
        keep = torch.rand(x.shape, generator=g, device=DEV) < 0.0005
        keep[:, 77] = True
        x.masked_fill_(~keep, -math.inf)
        tokens[:3] = 77
    elif case == "one_left":
        x.fill_(-math.inf)
        x[:, 12345] = torch.tensor([0.0, -3e38, 3e38, 5.0, -7.0, 1e-30], device=DEV)
        tokens[::2] = 12345
    elif case == "last":
        x[:, -1] = 50
        tokens.fill_(vocab - 1)
    elif case == "spread":
        x *= 1e4
    elif case == "zeros":  # -0 and +0 are equal
        x = torch.where(torch.rand(x.shape, generator=g, device=DEV) < 0.5, 0.0, -0.0)
    elif case == "huge_first":  # usual logits behind some that are far below them
        x[:, :vocab // 2] = -2e30
        tokens = tokens // 2 + vocab // 2
    elif case == "ascending":  # every next logit is a new maximum
        x = torch.arange(vocab, device=DEV).float().repeat(rows, 1) * 1e-2
    else:
        tokens = torch.tensor([-1, vocab, 2 ** 40, -2 ** 40, 0, vocab - 1], device=DEV)
    check_logprobs(x.to(dtype), tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_rows_without_a_finite_value(dtype):
    x = torch.randn(5, 5000, device=DEV).to(dtype)
    x[0] = -math.inf
    x[1, 4000] = math.nan
    x[2] = math.nan
    x[3, 17] = math.inf
    lp, ent, ids, tlp = kernels.token_logprobs(x, torch.zeros(5, dtype=torch.int64, device=DEV), 3)
    assert lp[0] == -math.inf and ent[0] == 0 and ids[0].tolist() == [0, 1, 2] and bool((tlp[0] == -math.inf).all())
    for r in (1, 2, 3):
        assert lp[r].isnan() and ent[r].isnan() and bool(tlp[r].isnan().all())
    assert 4000 not in ids[1].tolist() and ids[2].tolist() == [0, 1, 2] and ids[3, 0] == 17
    check_logprobs(x[4:], torch.tensor([3], device=DEV), 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_crowded_top(dtype):
    """Thousands of logits above what the rest of the row reaches, in a few columns of the 16-byte
    vectors; and thousands of ties at the last alternative, some in front of the larger logits."""
    g = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn(4, 151936, generator=g, device=DEV)
    column = torch.arange(151936, device=DEV) % 4096
    x[0, column < 64] += 100
    x[1, column < 32] += 100
    x[2] = torch.where(column < 2000, 7.0, x[2])
    x[2, 5000:5010] = torch.arange(8.0, 18.0, device=DEV)
    x[3, 100000:] = 3.0
    x[3, :100000].clamp_(max=2.0)
    for top in (2, 20, 32):
        check_logprobs(x.to(dtype), torch.tensor([3, 1, 2, 150000], device=DEV), top)
        check_logprobs(x.to(dtype).repeat(200, 1)[:, 1:], torch.randint(0, 151935, (800,), generator=g, device=DEV), top)


@pytest.mark.parametrize("vocab,nans", [(5, 3), (40, 20), (300, 299), (20011, 20000), (9000, 9000)])
def test_logprobs_nan_ranks_last(vocab, nans):
    g = torch.Generator(device=DEV).manual_seed(12)
    x = torch.randn(3, vocab, generator=g, device=DEV)
    x[:, torch.randperm(vocab, generator=g, device=DEV)[:nans]] = math.nan
    top = min(vocab, 32)
    _, _, ids, _ = kernels.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=DEV), top)
    key = torch.where(x.isnan(), -math.inf, x)
    assert torch.equal(ids, torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :top])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_strided_and_unaligned_rows(dtype):
    g = torch.Generator(device=DEV).manual_seed(10)
    wide = (torch.randn(9, 5003, generator=g, device=DEV) * 3).to(dtype)
    for lo, hi in ((1, 5000), (3, 5003), (0, 4999), (7, 8), (2, 1030)):
        check_logprobs(wide[:, lo:hi], torch.randint(0, hi - lo, (9,), generator=g, device=DEV), min(20, hi - lo))
        check_logprobs(wide[::2, lo:hi], torch.randint(0, hi - lo, (5,), generator=g, device=DEV), min(4, hi - lo))


def check_logprobs_of_any_size(x, tokens, top):
    """check_logprobs with a bound for logits of any size: the two 32-bit terms of a log probability, and
    of an entropy, are each up to 16 ln 2 < 12 beyond what is left of them (sums are kept relative to a
    logit of the row up to 11 below its maximum), with four roundings of 2^-24 of that and of x - m."""
    lp, ent, ids, tlp = kernels.token_logprobs(x, tokens, top)
    d = x.double()
    m = d.amax(-1, keepdim=True)
    y = torch.where(d == -math.inf, 0, d - m)
    e = torch.where(d == -math.inf, 0, torch.exp(d - m))
    z = e.sum(-1, keepdim=True)
    ln_z, spread, second = torch.log(z), (e * y.abs()).sum(-1, keepdim=True) / z, (e * y * y).sum(-1, keepdim=True) / z
    d_ln_z = (x.shape[1] / 1024 + 64) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * spread
    want = d - m - ln_z
    tol = d_ln_z + 2.0 ** -22 * ((d - m).abs() + ln_z + 12)
    at = tokens[:, None]
    close(lp, want.gather(1, at).squeeze(1), tol.gather(1, at).squeeze(1))
    close(ent, (ln_z + spread).squeeze(1), (d_ln_z * (1 + spread) + 2.0 ** -22 * (12 + second + spread + ln_z)).squeeze(1))
    order = torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ids, order)
    close(tlp, want.gather(1, order), tol.gather(1, order))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", [-3e4, -6e7, -1.01e8, -1e9, -1e10, -1e12, -1e20, -9.5e29, -1e30, -1e38, "lowest"])
def test_logprobs_of_rows_masked_with_a_finite_value(mask, dtype):
    """Guided decoding: most of a row at one low value; whole threads, blocks of a cluster and the row's
    ends see nothing else."""
    value = torch.finfo(dtype).min if mask == "lowest" else mask
    g = torch.Generator(device=DEV).manual_seed(60)
    for rows, vocab, top in ((1, 151936, 5), (6, 151937, 32), (300, 9001, 3), (320, 1003, 20)):
        x = (torch.randn(rows, vocab, generator=g, device=DEV) * 3).to(dtype)
        keep = torch.rand(rows, vocab, generator=g, device=DEV) < torch.tensor([0.1, 0.001, 0.5], device=DEV)[torch.arange(rows, device=DEV) % 3][:, None]
        keep[::2, :vocab // 2] = False
        keep[:, 3 * vocab // 4] = True
        tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        tokens[::2] = 3 * vocab // 4
        check_logprobs_of_any_size(x.masked_fill(~keep, value), tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("largest", [1e10, -1e10, 1e20, -1e20, 1e30, -9.5e29, -1e30, 3e38, -3e38, 5e7, -5e7, 2e8, -2e8])
def test_logprobs_of_rows_whose_maximum_is_large(largest, dtype):
    """Everything within a few steps of the type around one large value, the maximum a few times."""
    g = torch.Generator(device=DEV).manual_seed(61)
    for rows, vocab in ((2, 151936), (300, 3001)):
        steps = torch.randint(-9, 1, (rows, vocab), generator=g, device=DEV)
        steps[:, 7] = 0
        x = (largest + steps * (abs(largest) * torch.finfo(dtype).eps)).to(dtype)
        tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        tokens[0] = 7
        check_logprobs_of_any_size(x, tokens, 20)
        x[:, vocab // 3:] = -math.inf  # threads and blocks without a logit
        tokens %= vocab // 3
        check_logprobs_of_any_size(x, tokens, 20)


@pytest.mark.parametrize("middle", [-1e8, 1e8, -5e7, 5e7])
def test_logprobs_where_the_forms_of_the_exponent_meet(middle):
    """fp32 logits a few of their steps (4 or 8) apart on both sides of the sizes where a reference
    changes its form, sorted so that some threads see one side only."""
    g = torch.Generator(device=DEV).manual_seed(62)
    for rows, vocab in ((1, 151936), (40, 20011), (300, 1500)):
        x = (middle + 8.0 * torch.randint(-9, 9, (rows, vocab), generator=g, device=DEV)).float()
        x[:, vocab // 2:] = x[:, vocab // 2:].sort(-1).values
        x[::2] = x[::2].flip(1)
        check_logprobs_of_any_size(x, torch.randint(0, vocab, (rows,), generator=g, device=DEV), 8)


@pytest.mark.parametrize("rows", [1, 149, 600])
def test_logprobs_of_large_logits_one_step_of_fp32_apart(rows):
    """Most of a row at 2e8, some a step of 16 above it: the reference has to be the row's maximum."""
    g = torch.Generator(device=DEV).manual_seed(65)
    x = 2e8 + 16.0 * (torch.rand(rows, 77412, generator=g, device=DEV) < 0.0036)
    check_logprobs_of_any_size(x, torch.randint(0, 77412, (rows,), generator=g, device=DEV), 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_are_never_positive_and_entropies_never_negative(dtype):
    """Confident rows, whose own token is nearly certain."""
    g = torch.Generator(device=DEV).manual_seed(63)
    for rows, vocab in ((256, 20011), (1000, 3001), (2, 151936)):
        x = (torch.randn(rows, vocab, generator=g, device=DEV) * 2.5).to(dtype)
        tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        x.scatter_(1, tokens[:, None], (20 + 25 * torch.rand(rows, 1, generator=g, device=DEV)).to(dtype))
        lp, ent, ids, tlp = kernels.token_logprobs(x, tokens, 3)
        assert bool((lp <= 0).all()) and bool((tlp <= 0).all()) and bool((ent >= 0).all())
        check_logprobs_of_any_size(x, tokens, 3)


def test_logprobs_rows_behind_4_gib():
    x = torch.zeros(9000, 262144, dtype=torch.bfloat16, device=DEV)
    x[:, 5] = 3
    lp, ent, ids, _ = kernels.token_logprobs(x, torch.full((9000,), 5, device=DEV), 1)
    assert bool((ids == 5).all()) and lp.unique().numel() == 1 and ent.unique().numel() == 1
    assert abs(float(lp[-1]) - (3 - math.log(262143 + math.exp(3)))) < 1e-5


# ----------------------------------------------------------------------------- together
def test_a_prompt_and_decode_steps_through_all_operators_in_a_graph():
    """Prompts get pages and are stored; then decode steps, captured once and replayed: tables,
    store, attention, a projection to logits, sampling, log probabilities."""
    g = torch.Generator().manual_seed(30)
    hq, hk, bs, t, nb, vocab, steps = 8, 4, 256, 64, 40, 1003, 3
    lens = [5, 256, 300, 63, 0]  # the last one is a padding slot
    b, width = len(lens), 3
    i32 = dict(dtype=torch.int32, device=DEV)
    caches = torch.zeros(2, nb, bs, hk, D, dtype=torch.uint8, device=DEV).view(E4M3)
    scales = torch.zeros(2, nb, bs // t, hk, device=DEV)
    ref = [[c.cpu(), s.cpu()] for c, s in zip(caches.float().to(E4M3), scales)]
    tables = torch.full((b, width), -1, **i32)
    free = torch.randperm(nb, generator=g).int().to(DEV)
    prompt = torch.randn(2, sum(lens), hk, D, generator=g).bfloat16()
    plan = kernels.extend_block_tables(tables, None, torch.tensor(lens, **i32), free, bs, sum(lens) + 4)
    assert plan["status"][1] == 0
    taken = int(plan["status"][0])
    kernels.store_kvcache_fp8_blocks(prompt[0].to(DEV), prompt[1].to(DEV), caches[0], caches[1], scales[0], scales[1],
                                     tables, plan["context_lens"], plan["cu_seqlens_q"])
    cu = np.concatenate(([0], np.cumsum(lens))).tolist()
    for x, (c, s) in zip(prompt, ref):
        store_ref(x, c, s, tables.tolist(), lens, cu)

    qkv = torch.randn(steps, b, hq + 2 * hk, D, generator=g).bfloat16()
    head = (torch.randn(hq * D, vocab, generator=g) / 10).bfloat16().to(DEV)
    live = torch.tensor([1, 1, 1, 1, 0], **i32)
    cached, pages_left, row_in = torch.tensor(lens, **i32), free[taken:].clone(), torch.empty_like(qkv[0], device=DEV)
    ws = kernels.make_block_decode_workspace(b, hq, hk, torch.device(DEV))

    def step():
        plan = kernels.extend_block_tables(tables, cached, live, pages_left, bs, b)
        kernels.store_kvcache_fp8_blocks(row_in[:, hq:hq + hk], row_in[:, hq + hk:], caches[0], caches[1], scales[0], scales[1],
                                         tables, plan["context_lens"], plan["cu_seqlens_q"])
        out = kernels.paged_decode_fp8_blocks(row_in[:, :hq], caches[0], caches[1], scales[0], scales[1], tables,
                                              plan["context_lens"], D ** -0.5, workspace=ws)
        logits = out.view(b, -1) @ head
        tokens = kernels.sample(logits, None, 0, None)
        return plan, out, logits, tokens, kernels.token_logprobs(logits, tokens, 4)

    saved = [x.clone() for x in (tables, caches.view(torch.uint8), scales)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up, then capture
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, out, logits, tokens, (lp, ent, ids, tlp) = step()
    for x, y in zip((tables, caches.view(torch.uint8), scales), saved):
        x.copy_(y)
    now = list(lens)
    for k in range(steps):
        row_in.copy_(qkv[k])
        cached.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        now = [n + int(a) for n, a in zip(now, live.tolist())]
        used = int(plan["status"][0])
        pages_left.copy_(torch.roll(pages_left, -used))
        assert plan["status"][1] == 0 and plan["context_lens"].tolist() == now
        cu = [0, 1, 2, 3, 4, 4]
        store_ref(qkv[k][:, hq:hq + hk], *ref[0], tables.tolist(), now, cu)
        store_ref(qkv[k][:, hq + hk:], *ref[1], tables.tolist(), now, cu)
        for i in range(2):
            assert same_bytes(caches[i], ref[i][0]) and torch.equal(scales[i].cpu(), ref[i][1])
        want, mass, size = decode_ref(row_in[:, :hq], caches[0], caches[1], scales[0], scales[1], tables.tolist(), now, D ** -0.5)
        tol = want.abs() * 2.0 ** -8 + mass * (2.0 ** -11 + 2.0 ** -18 + 2 * 130 * 2.0 ** -23 * size) + 1e-37
        assert bool(((out.double() - want).abs() <= tol).all()) and not out[4].any()
        assert torch.equal(tokens, ids[:, 0])
        full = torch.log_softmax(logits.double(), -1)
        assert bool(((lp.double() - full.gather(1, tokens[:, None]).squeeze(1)).abs() < 1e-5).all())
        assert torch.equal(lp, tlp[:, 0]) and bool(((ent.double() + (full.exp() * full).sum(-1)).abs() < 1e-5).all())
    assert kernels.decode_errors(ws) == 0


def test_two_streams_with_a_workspace_each():
    a, c = decode_case(41, 8, 4, 256, 64, [20000, 7]), decode_case(42, 8, 2, 256, 64, [900] * 60)
    i32 = dict(dtype=torch.int32, device=DEV)
    args = [[*x[:5], torch.tensor(x[5], **i32), torch.tensor(x[6], **i32), 0.09] for x in (a, c)]
    spaces = [kernels.make_block_decode_workspace(x[0].shape[0], x[0].shape[1], 8, x[0].device) for x in (a, c)]
    want = [kernels.paged_decode_fp8_blocks(*x, workspace=w) for x, w in zip(args, spaces)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kernels.paged_decode_fp8_blocks(*args[i], workspace=spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_calls_queued_behind_each_other_keep_the_streams_order():
    """Steps that each read what the one before wrote, without a wait between them, against the same
    steps with one after every call."""
    g = torch.Generator(device=DEV).manual_seed(50)
    hq, hk, bs, t, nb, b, vocab, steps = 8, 2, 256, 64, 30, 9, 2000, 70
    qkv = torch.randn(steps, b, hq + 2 * hk, D, generator=g, device=DEV).bfloat16() * torch.logspace(
        -2, 2, steps, device=DEV).view(-1, 1, 1, 1).bfloat16()
    head = torch.randn(hq * D, vocab, generator=g, device=DEV).bfloat16()
    i32 = dict(dtype=torch.int32, device=DEV)
    start = torch.tensor([0, 1, 62, 63, 64, 150, 180, 300, 400], **i32)  # nobody needs a new page, which would be free[0] each time
    free = torch.arange(nb, **i32)

    def run(wait):
        pause = torch.cuda.synchronize if wait else lambda: None
        caches = torch.zeros(2, nb, bs, hk, D, dtype=torch.uint8, device=DEV).view(E4M3)
        scales = torch.zeros(2, nb, bs // t, hk, device=DEV)
        tables, seen = torch.full((b, 3), -1, **i32), []
        kernels.extend_block_tables(tables, None, torch.full((b,), 500, **i32), free, bs, 0)
        ws, context = kernels.make_block_decode_workspace(b, hq, hk, torch.device(DEV)), start
        for x in qkv:
            plan = kernels.extend_block_tables(tables, context, torch.ones(b, **i32), free, bs, b)
            pause()
            context = plan["context_lens"]
            kernels.store_kvcache_fp8_blocks(x[:, hq:hq + hk], x[:, hq + hk:], caches[0], caches[1], scales[0], scales[1],
                                             tables, context, plan["cu_seqlens_q"])
            pause()
            out = kernels.paged_decode_fp8_blocks(x[:, :hq], caches[0], caches[1], scales[0], scales[1], tables, context,
                                                  D ** -0.5, workspace=ws)
            pause()
            logits = out.view(b, -1) @ head
            pause()
            seen += [out, *kernels.token_logprobs(logits, plan["positions"] % vocab, 3), plan["slot_mapping"]]
            pause()
        return seen + [caches.view(torch.uint8), scales, tables]

    for got, want in zip(run(False), run(True)):
        assert torch.equal(got, want)


def test_captured_behind_copies_fills_and_joined_branches():
    """Graphs whose launches follow a memset, a copy or two branches of the capture, and two graphs that use
    one workspace in turn."""
    g = torch.Generator(device=DEV).manual_seed(74)
    q, kc, vc, ks, vs, tables, context = decode_case(75, 4, 4, 256, 64, [3000, 1, 700, 0, 65])
    i32 = dict(dtype=torch.int32, device=DEV)
    tables, context = torch.tensor(tables, **i32), torch.tensor(context, **i32)
    x = torch.randn(5, 2, 4, D, generator=g, device=DEV).bfloat16()
    logits = torch.randn(5, 20011, generator=g, device=DEV).bfloat16()
    tokens, free = torch.arange(5, device=DEV), torch.arange(50, **i32)
    ws = kernels.make_block_decode_workspace(5, 16, 4, q.device)
    start = [t.clone() for t in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    state = (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)
    ones = torch.ones(5, **i32)

    def step(workspace, split):
        main, side = torch.cuda.current_stream(), torch.cuda.Stream()
        table = torch.full_like(tables, -1)                      # a fill in front of the table kernel
        plan = kernels.extend_block_tables(table, None, ones, free, 256, 8)
        if split:
            side.wait_stream(main)
            with torch.cuda.stream(side):
                lp = kernels.token_logprobs(logits, tokens, 4)
            kernels.store_kvcache_fp8_blocks(x[:, 0], x[:, 1], kc, vc, ks, vs, tables, context)
            main.wait_stream(side)                               # two branches in front of the attention
        else:
            kernels.store_kvcache_fp8_blocks(x[:, 0], x[:, 1], kc, vc, ks, vs, tables, context)
            lp = kernels.token_logprobs(logits, tokens, 4)
        out = kernels.paged_decode_fp8_blocks(q, kc, vc, ks, vs, tables, context, D ** -0.5, workspace=workspace)
        copied = out.clone()                                     # a copy in front of the next call
        return [plan["slot_mapping"], table, *lp, copied, *kernels.token_logprobs(copied.view(5, -1), tokens, 3)]

    want = [t.clone() for t in step(ws, False)]
    after = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(None, True)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for workspace, split in ((ws, True), (ws, False), (None, True)):  # None: its fill is part of the graph
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(workspace, split)
        graphs.append((graph, out))
    for _ in range(3):
        for graph, out in graphs:
            for t, s in zip(state, start):
                t.copy_(s)
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert all(torch.equal(a, b) for a, b in zip(state, after))
    assert kernels.decode_errors(ws) == 0
