"""What the serving operators refuse, at the C ABI and in the Python wrappers; no GPU needed: every
check comes before the first launch."""
import ctypes

import pytest
import torch

from hilda_vllm_b200 import _lib, kernels

P = ctypes.c_void_p(256)      # aligned, never dereferenced by a refused call
ODD = ctypes.c_void_p(8)


def call(name, args, changed, status=1, text=""):
    args = dict(args)
    for k in changed:
        assert k in args
    args.update(changed)
    lib = _lib.load()
    assert getattr(lib, name)(*args.values(), None) == status
    assert text.encode() in lib.hl_last_error_string()


TABLES = dict(cached=P, query=P, seqs=4, tables=P, stride=8, width=8, free=P, num_free=9, bs=256, tokens=10, cu_q=P, cu_k=P,
              ctx=P, pos=P, slots=P, status=P)


@pytest.mark.parametrize("changed,text", [
    ({"seqs": -1}, "num_seqs"), ({"seqs": 4097}, "num_seqs"), ({"bs": 0}, "block_size"), ({"width": 0}, "width"),
    ({"stride": 7}, "width"), ({"num_free": -1}, "num_free"), ({"tokens": -1}, "max_tokens"), ({"tokens": 1 << 31}, "max_tokens"),
    ({"query": None}, "null"), ({"free": None}, "null"), ({"slots": None}, "null"), ({"status": None}, "null"),
])
def test_tables_refusals(changed, text):
    call("hl_extend_block_tables", TABLES, changed, text=text)


@pytest.mark.parametrize("result", ["cu_q", "cu_k", "ctx", "pos", "slots", "status"])
@pytest.mark.parametrize("given,entries", [("cached", 4), ("query", 4), ("free", 9)])
def test_tables_refuse_results_that_overwrite_what_is_read(result, given, entries):
    """Among them context_lens == cached_lens: all blocks read the lengths while the first writes."""
    apart = {k: ctypes.c_void_p(4096 * (i + 1)) for i, k in enumerate(("cached", "query", "tables", "free", "cu_q", "cu_k", "ctx", "pos",
                                                                       "slots", "status"))}
    sizes = dict(cu_q=20, cu_k=20, ctx=16, pos=80, slots=40, status=8)
    first = apart[given].value
    for at in (first, first + 4 * entries - 4, first - sizes[result] + 4):
        call("hl_extend_block_tables", TABLES, {**apart, result: ctypes.c_void_p(at)}, text="overlaps")


STORE = dict(key=P, value=P, krs=1024, vrs=1024, tokens=5, kc=P, vc=P, ks=P, vs=P, tables=P, stride=4, width=4, ctx=P, cu=P, seqs=3,
             hk=8, d=128, bs=256, t=64, nb=10)


@pytest.mark.parametrize("changed,text", [
    ({"tokens": -1}, "num_tokens"), ({"seqs": -1}, "num_seqs"), ({"d": 64}, "head_dim"), ({"hk": 0}, "num_kv_heads"),
    ({"t": 32}, "scale_block"), ({"t": 96}, "scale_block"), ({"t": 512}, "scale_block"), ({"t": 0}, "scale_block"),
    ({"bs": 0}, "scale_block"), ({"cu": None}, "one token per sequence"), ({"value": None}, "null"), ({"ks": None}, "null"),
    ({"width": 5}, "block table"), ({"nb": 0}, "pool"), ({"krs": 1016}, "stride"), ({"key": ODD}, "alignment"),
    ({"vrs": 1028}, "alignment"), ({"vc": ODD}, "alignment"),
])
def test_store_refusals(changed, text):
    call("hl_store_kv_fp8_blocks", STORE, changed, text=text)


DECODE = dict(q=P, qrs=2048, kc=P, vc=P, ks=P, vs=P, tables=P, stride=4, width=4, ctx=P, batch=3, hq=16, hk=8, d=128, bs=256, t=64,
              nb=10, scale=0.1, out=P, ors=2048, ws=P, ws_bytes=1 << 30)


@pytest.mark.parametrize("changed,text", [
    ({"batch": -1}, "batch"), ({"batch": 4097}, "batch"), ({"d": 64}, "head_dim"), ({"hq": 12}, "multiple"), ({"hq": 136}, "16 query"),
    ({"hk": 0}, "multiple"), ({"t": 32}, "scale_block"), ({"bs": 250}, "scale_block"), ({"nb": 0}, "pool"), ({"width": 5}, "block table"),
    ({"width": 1 << 23, "stride": 1 << 23}, "2^31"), ({"q": None}, "null"), ({"vs": None}, "null"), ({"q": ODD}, "alignment"),
    ({"qrs": 2047}, "alignment"), ({"ors": 2040}, "alignment"), ({"kc": ODD}, "alignment"),
])
def test_decode_refusals(changed, text):
    call("hl_paged_decode_fp8_blocks", DECODE, changed, text=text)


def test_decode_workspace():
    lib = _lib.load()
    call("hl_paged_decode_fp8_blocks", DECODE, {"ws": None}, 4, "workspace")
    call("hl_paged_decode_fp8_blocks", DECODE, {"ws_bytes": 16}, 4, "workspace")
    call("hl_paged_decode_fp8_blocks", DECODE, {"ws": ODD}, 4, "workspace")
    size = lib.hl_paged_decode_fp8_blocks_workspace_size
    assert size(0, 16, 8) == size(4, 12, 8) == size(4, 16, 0) == size(4097, 16, 8) == -1
    assert 0 < size(1, 16, 8) <= size(256, 16, 8) <= size(256, 32, 8)


LOGPROBS = dict(logits=P, fp32=0, stride=1000, rows=4, vocab=1000, tokens=P, top=5, lp=P, ent=P, ids=P, tlp=P)


@pytest.mark.parametrize("changed,text", [
    ({"rows": -1}, "shape"), ({"vocab": 0}, "shape"), ({"stride": 999}, "shape"), ({"top": -1}, "top_n"), ({"top": 33}, "top_n"),
    ({"top": 5, "vocab": 4, "stride": 4}, "top_n"), ({"logits": None}, "null"), ({"tokens": None}, "null"), ({"ids": None}, "null"),
    ({"ent": None}, "null"),
])
def test_logprobs_refusals(changed, text):
    call("hl_token_logprobs", LOGPROBS, changed, text=text)


def test_empty_calls_succeed_without_a_gpu():
    call("hl_store_kv_fp8_blocks", STORE, {"tokens": 0, "key": None}, 0)
    call("hl_paged_decode_fp8_blocks", DECODE, {"batch": 0, "q": None}, 0)
    call("hl_token_logprobs", LOGPROBS, {"rows": 0, "logits": None}, 0)


def test_wrappers_refuse_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    cache, scales = torch.zeros(2, 256, 8, 128).to(torch.float8_e4m3fn), torch.ones(2, 4, 8)
    for refused in (lambda: kernels.extend_block_tables(i.view(2, 1), i, i, i, 256, 2),
                    lambda: kernels.store_kvcache_fp8_blocks(x, x, cache, cache, scales, scales, i.view(2, 1), i),
                    lambda: kernels.paged_decode_fp8_blocks(x, cache, cache, scales, scales, i.view(2, 1), i, 0.1),
                    lambda: kernels.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError, match="no CPU fallback"):
            refused()


def test_wrappers_check_the_cache_shapes():
    cache, scales = torch.zeros(2, 256, 8, 128).to(torch.float8_e4m3fn), torch.ones(2, 4, 8)
    assert kernels._check_block_cache(cache, cache, scales, scales) == (2, 256, 8, 128, 64)
    for bad in ((cache.float(), cache, scales, scales), (cache, cache[:1], scales, scales), (cache, cache, scales[:, :3], scales[:, :3]),
                (cache, cache, scales.double(), scales), (cache, cache, scales[:, :, :4], scales[:, :, :4]),
                (cache.transpose(1, 2), cache.transpose(1, 2), scales, scales), (cache, cache, scales, scales[:1])):
        with pytest.raises(AssertionError):
            kernels._check_block_cache(*bad)
