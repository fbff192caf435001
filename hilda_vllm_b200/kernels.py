"""PyTorch-facing wrappers of the C ABI (include/hilda_b200.h).

Each wrapper validates shapes the way the reference does (mini_vllm/layers/attention.py:83-90
asserts strides), passes raw device pointers and the current CUDA stream to the library and
raises HildaKernelError on a non-zero status.  Tensors must live on a CUDA device; there is
no CPU path.  Every call only launches kernels on the current stream, so all of them can be
captured in a CUDA graph (workspaces are caller-provided or created before capture).
"""
from __future__ import annotations

import ctypes

import torch

from hilda_vllm_b200 import _lib
from hilda_vllm_b200._lib import HlPackEvent, HlPackHeader, check

KV_BF16 = 0
KV_FP8_E4M3 = 1

# Flags of hl_pack_event (include/hilda_b200.h).
EV_SCALARS = 1
EV_ROW = 2
EV_ROW_FILL = 4
EV_CLEAR = 8


def _cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("hilda_vllm_b200 kernels need CUDA tensors (there is no CPU fallback)")


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _p(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# ----------------------------------------------------------------------------- KV store
def _check_store_args(key, value, k_cache, v_cache, slot_mapping):
    n, num_heads, head_dim = key.shape
    d = num_heads * head_dim
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert k_cache.stride(1) == d and v_cache.stride(1) == d
    assert slot_mapping.numel() == n
    assert slot_mapping.dtype == torch.int32 and slot_mapping.is_contiguous()
    assert key.dtype == torch.bfloat16 and value.dtype == torch.bfloat16
    _cuda(key, value, k_cache, v_cache, slot_mapping)
    return n, num_heads, head_dim


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slot_mapping: torch.Tensor) -> None:
    """BF16 scatter of key/value [N, Hk, D] into k_cache/v_cache [NB, BS, Hk, D] by slot_mapping
    (slot -1 skipped).  Same contract as mini_vllm/layers/attention.py:83-90."""
    n, hk, hd = _check_store_args(key, value, k_cache, v_cache, slot_mapping)
    assert k_cache.dtype == torch.bfloat16 and v_cache.dtype == torch.bfloat16
    if n == 0:
        return
    num_slots = k_cache.shape[0] * k_cache.shape[1]
    lib = _lib.load()
    check(lib.hl_store_kv_bf16(key.data_ptr(), value.data_ptr(), key.stride(0), value.stride(0),
                               k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), n, num_slots,
                               hk, hd, _stream(key)), "hl_store_kv_bf16")


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slot_mapping: torch.Tensor, k_scale: torch.Tensor | None = None,
                      v_scale: torch.Tensor | None = None) -> None:
    """BF16 -> FP8 e4m3 quantising store with per-KV-head fp32 scales (None = unit scale,
    the reference's hilda_store_kvcache_fp8 signature, attention.py:51-52)."""
    n, hk, hd = _check_store_args(key, value, k_cache, v_cache, slot_mapping)
    assert k_cache.dtype == torch.float8_e4m3fn and v_cache.dtype == torch.float8_e4m3fn
    for s in (k_scale, v_scale):
        if s is not None:
            assert s.dtype == torch.float32 and s.numel() == hk and s.is_contiguous()
    _cuda(k_scale, v_scale)
    if n == 0:
        return
    num_slots = k_cache.shape[0] * k_cache.shape[1]
    lib = _lib.load()
    check(lib.hl_store_kv_fp8(key.data_ptr(), value.data_ptr(), key.stride(0), value.stride(0),
                              k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), n, num_slots,
                              hk, hd, _p(k_scale), _p(v_scale), _stream(key)), "hl_store_kv_fp8")


def copy_kvcache_fp8(src_k_cache: torch.Tensor, src_v_cache: torch.Tensor, dst_k_cache: torch.Tensor,
                     dst_v_cache: torch.Tensor, slot_mapping: torch.Tensor, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> None:
    """One layer: dst[slot] = fp8(src[slot] / scale) for every slot in slot_mapping
    (the reference's copy_kvcache_fp8, attention.py:55-56)."""
    copy_kvcache_fp8_layers(src_k_cache.unsqueeze(0), src_v_cache.unsqueeze(0), dst_k_cache.unsqueeze(0),
                            dst_v_cache.unsqueeze(0), slot_mapping,
                            None if k_scale is None else k_scale.view(1, -1),
                            None if v_scale is None else v_scale.view(1, -1))


def copy_kvcache_fp8_layers(src_k: torch.Tensor, src_v: torch.Tensor, dst_k: torch.Tensor, dst_v: torch.Tensor,
                            slot_mapping: torch.Tensor, k_scales: torch.Tensor | None = None,
                            v_scales: torch.Tensor | None = None) -> None:
    """All layers in one launch: src_* [L, NB, BS, Hk, D] bf16, dst_* same shape e4m3,
    k_scales/v_scales [L, Hk] fp32 (or None)."""
    _cuda(src_k, src_v, dst_k, dst_v, slot_mapping, k_scales, v_scales)
    num_layers, nb, bs, hk, hd = src_k.shape
    assert src_k.dtype == torch.bfloat16 and dst_k.dtype == torch.float8_e4m3fn
    assert src_k.stride() == src_v.stride() and dst_k.stride() == dst_v.stride()
    assert src_k.stride(1) == bs * hk * hd and dst_k.stride(1) == bs * hk * hd
    assert src_k.stride()[2:] == (hk * hd, hd, 1) and dst_k.stride()[2:] == (hk * hd, hd, 1)
    assert slot_mapping.dtype == torch.int32 and slot_mapping.is_contiguous()
    scale_stride = 0
    for s in (k_scales, v_scales):
        if s is not None:
            assert s.dtype == torch.float32 and s.shape == (num_layers, hk) and s.is_contiguous()
            scale_stride = hk
    n = slot_mapping.numel()
    if n == 0:
        return
    lib = _lib.load()
    check(lib.hl_copy_kv_bf16_to_fp8(src_k.data_ptr(), src_v.data_ptr(), dst_k.data_ptr(), dst_v.data_ptr(),
                                     slot_mapping.data_ptr(), n, nb * bs, hk, hd, _p(k_scales), _p(v_scales),
                                     num_layers, src_k.stride(0), dst_k.stride(0), scale_stride,
                                     _stream(src_k)), "hl_copy_kv_bf16_to_fp8")


# ------------------------------------------------------------------------ decode attention
def decode_workspace_bytes(batch: int, num_q_heads: int, head_dim: int, max_blocks_per_seq: int,
                           block_size: int) -> int:
    n = _lib.load().hl_paged_decode_workspace_size(batch, num_q_heads, head_dim, max_blocks_per_seq, block_size)
    if n < 0:
        raise ValueError("bad decode workspace shape")
    return int(n)


def make_decode_workspace(batch: int, num_q_heads: int, head_dim: int, max_blocks_per_seq: int,
                          block_size: int, device) -> torch.Tensor:
    """Zero-filled workspace for paged_decode (its tickets must start at zero)."""
    n = decode_workspace_bytes(batch, num_q_heads, head_dim, max_blocks_per_seq, block_size)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, softmax_scale: float, out: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, tensor_cores: bool = False) -> torch.Tensor:
    """Decode attention for one new token per sequence over the paged cache.

    q [B, Hq, D] (or [B, 1, Hq, D]) bf16; k_cache/v_cache [NB, BS, Hk, D] bf16 or e4m3;
    block_tables [B, >= max_blocks] int32; context_lens [B] int32.  Returns out [B, Hq, D].
    The semantics are flash_attn_with_kvcache's for a single causal query token
    (mini_vllm/layers/attention.py:162-170).  The library picks the kernel (the tcgen05 one for
    GQA ratios >= 4); tensor_cores=True forces the tcgen05 variant (hl_paged_decode_tc) for any
    ratio it supports."""
    if q.dim() == 4:
        assert q.shape[1] == 1
        q = q.squeeze(1)
    _cuda(q, k_cache, v_cache, block_tables, context_lens, out, workspace, k_scale, v_scale)
    b, hq, hd = q.shape
    nb, bsz, hk, hd2 = k_cache.shape
    assert hd == hd2 and q.stride(2) == 1 and q.stride(1) == hd
    assert k_cache.is_contiguous() and v_cache.is_contiguous() and v_cache.shape == k_cache.shape
    assert block_tables.dtype == torch.int32 and block_tables.stride(1) == 1 and block_tables.shape[0] >= b
    assert context_lens.dtype == torch.int32 and context_lens.is_contiguous() and context_lens.numel() >= b
    if k_cache.dtype == torch.bfloat16:
        kv_dtype = KV_BF16
    elif k_cache.dtype == torch.float8_e4m3fn:
        kv_dtype = KV_FP8_E4M3
    else:
        raise TypeError(f"unsupported cache dtype {k_cache.dtype}")
    if out is None:
        out = torch.empty(b, hq, hd, dtype=torch.bfloat16, device=q.device)
    assert out.dtype == torch.bfloat16 and out.stride(2) == 1 and out.stride(1) == hd
    if b == 0:
        return out
    max_blocks = block_tables.shape[1]
    if workspace is None:
        workspace = make_decode_workspace(b, hq, hd, max_blocks, bsz, q.device)
    lib = _lib.load()
    fn = lib.hl_paged_decode_tc if tensor_cores else lib.hl_paged_decode
    check(fn(q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), kv_dtype,
             _p(k_scale), _p(v_scale), block_tables.data_ptr(), block_tables.stride(0),
             max_blocks, context_lens.data_ptr(), b, hq, hk, hd, bsz, nb, float(softmax_scale),
             out.data_ptr(), out.stride(0), workspace.data_ptr(), workspace.numel(),
             _stream(q)), "hl_paged_decode")
    return out


def decode_errors(workspace: torch.Tensor) -> int:
    """Error bits the decode kernel recorded in its workspace (synchronises the stream)."""
    val = ctypes.c_int32(0)
    check(_lib.load().hl_paged_decode_read_errors(workspace.data_ptr(), ctypes.addressof(val), _stream(workspace)),
          "hl_paged_decode_read_errors")
    return int(val.value)


# ------------------------------------------------------------------------ prefill attention
def varlen_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                   cu_seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int, softmax_scale: float,
                   block_table: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   precise_p: bool = True, one_head_per_cta: bool = False) -> torch.Tensor:
    """Causal varlen attention with a bottom-right-aligned mask on the tcgen05/TMEM kernel.

    Same arguments as the reference's flash_attn_varlen_func call
    (mini_vllm/layers/attention.py:149-160): q [Tq, Hq, D]; with block_table, k/v are the paged
    caches [NB, BS, Hk, D]; without, k/v are [Tk, Hk, D].  Returns [Tq, Hq, D] bf16.
    precise_p feeds P to the P.V MMA as bf16 hi + lo terms (see hl_varlen_prefill);
    one_head_per_cta forces the one-query-head-per-CTA kernel instead of the head-pair kernel."""
    _cuda(q, k, v, cu_seqlens_q, cu_seqlens_k, block_table, out)
    tq, hq, hd = q.shape
    assert q.stride(2) == 1 and q.stride(1) == hd
    assert cu_seqlens_q.dtype == torch.int32 and cu_seqlens_k.dtype == torch.int32
    num_seqs = cu_seqlens_q.numel() - 1
    if block_table is not None:
        nb, bsz, hk, _ = k.shape
        assert k.is_contiguous() and v.is_contiguous()
        assert block_table.dtype == torch.int32 and block_table.stride(1) == 1
        bt_ptr, bt_stride, k_rs, v_rs, total_k = block_table.data_ptr(), block_table.stride(0), 0, 0, 0
    else:
        total_k, hk, _ = k.shape
        assert k.stride(2) == 1 and k.stride(1) == hd and v.stride(2) == 1 and v.stride(1) == hd
        nb, bsz = 0, 0
        bt_ptr, bt_stride, k_rs, v_rs = None, 0, k.stride(0), v.stride(0)
    if out is None:
        out = torch.empty(tq, hq, hd, dtype=torch.bfloat16, device=q.device)
    if num_seqs <= 0 or tq == 0:
        return out
    lib = _lib.load()
    check(lib.hl_varlen_prefill(q.data_ptr(), q.stride(0), tq, k.data_ptr(), v.data_ptr(), k_rs, v_rs, total_k,
                                   cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), bt_ptr, bt_stride, num_seqs,
                                   int(max_seqlen_q), hq, hk, hd, bsz, nb, float(softmax_scale), out.data_ptr(),
                                   out.stride(0), (1 if precise_p else 0) | (2 if one_head_per_cta else 0),
                                   _stream(q)), "hl_varlen_prefill")
    return out


def prefill_errors() -> int:
    """Error bits of the tensor-core prefill kernel (synchronous)."""
    val = ctypes.c_int32(0)
    check(_lib.load().hl_varlen_prefill_read_errors(ctypes.addressof(val)), "hl_varlen_prefill_read_errors")
    return int(val.value)


def copy_prefill_errors_async(dst: torch.Tensor) -> None:
    """Queues a copy of the prefill kernel's error word into dst (an int32 element of pinned host
    or device memory) on the current stream."""
    assert dst.dtype == torch.int32 and dst.numel() >= 1
    check(_lib.load().hl_varlen_prefill_copy_errors_async(dst.data_ptr(), torch.cuda.current_stream().cuda_stream),
          "hl_varlen_prefill_copy_errors_async")


# ------------------------------------------------------------------------ decode packing
def pack_decode_batch(packet: torch.Tensor, graph_batch: int, block_size: int, slot_seq_ids: torch.Tensor,
                      slot_bt_lens: torch.Tensor, next_tokens: torch.Tensor, input_ids: torch.Tensor,
                      positions: torch.Tensor, slot_mapping: torch.Tensor, context_lens: torch.Tensor,
                      block_tables: torch.Tensor) -> None:
    """Rebuilds the persistent decode buffers on the device from the packet (a device uint8
    buffer: hl_pack_header, events, block-id pool; see hl_pack_decode_batch)."""
    _cuda(packet, slot_seq_ids, slot_bt_lens, next_tokens, input_ids, positions, slot_mapping, context_lens,
          block_tables)
    assert packet.dtype == torch.uint8 and packet.is_contiguous()
    assert block_tables.dtype == torch.int32 and block_tables.stride(1) == 1
    assert slot_seq_ids.dtype == torch.int64 and slot_bt_lens.dtype == torch.int32
    assert input_ids.dtype == torch.int64 and positions.dtype == torch.int64 and next_tokens.dtype == torch.int64
    assert slot_mapping.dtype == torch.int32 and context_lens.dtype == torch.int32
    lib = _lib.load()
    check(lib.hl_pack_decode_batch(packet.data_ptr(), packet.numel(), int(graph_batch), int(block_size),
                                   slot_seq_ids.data_ptr(), slot_bt_lens.data_ptr(), next_tokens.data_ptr(),
                                   input_ids.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(),
                                   context_lens.data_ptr(), block_tables.data_ptr(), block_tables.stride(0),
                                   block_tables.shape[1], _stream(block_tables)), "hl_pack_decode_batch")


PACK_EVENT_BYTES = ctypes.sizeof(HlPackEvent)
PACK_HEADER_BYTES = ctypes.sizeof(HlPackHeader)


# ------------------------------------------------------------------------ layer kernels
def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None,
            out: torch.Tensor | None = None):
    """RMSNorm (residual None) or add+RMSNorm updating `residual` in place; returns out or
    (out, residual) like RMSNorm.forward (mini_vllm/layers/layernorm.py:44-52)."""
    _cuda(x, weight, residual, out)
    rows, hidden = x.shape
    assert x.stride(1) == 1 and weight.is_contiguous()
    if out is None:
        out = torch.empty(rows, hidden, dtype=x.dtype, device=x.device)
    if residual is not None:
        assert residual.is_contiguous() and residual.shape == x.shape
    lib = _lib.load()
    check(lib.hl_rmsnorm(x.data_ptr(), x.stride(0), _p(residual), weight.data_ptr(), out.data_ptr(), out.stride(0),
                         rows, hidden, float(eps), _stream(x)), "hl_rmsnorm")
    return out if residual is None else (out, residual)


def qk_norm_rope(qkv: torch.Tensor, num_q_heads: int, num_kv_heads: int, head_dim: int, q_weight: torch.Tensor,
                 k_weight: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor, eps: float) -> None:
    """In place on qkv [T, (Hq+2Hk)*D]: per-head RMSNorm of q and k, then NeoX RoPE."""
    _cuda(qkv, q_weight, k_weight, cos_sin, positions)
    assert qkv.stride(1) == 1 and cos_sin.dtype == torch.float32 and cos_sin.is_contiguous()
    assert positions.dtype == torch.int64 and positions.is_contiguous()
    lib = _lib.load()
    check(lib.hl_qk_norm_rope(qkv.data_ptr(), qkv.stride(0), qkv.shape[0], num_q_heads, num_kv_heads, head_dim,
                              q_weight.data_ptr(), k_weight.data_ptr(), cos_sin.data_ptr(), positions.data_ptr(),
                              float(eps), _stream(qkv)), "hl_qk_norm_rope")


def qk_norm_rope_store(qkv: torch.Tensor, num_q_heads: int, num_kv_heads: int, head_dim: int,
                       q_weight: torch.Tensor, k_weight: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor,
                       eps: float, k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                       k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                       k_mirror: torch.Tensor | None = None, v_mirror: torch.Tensor | None = None) -> None:
    """qk_norm_rope plus the KV-cache store of the rotated k heads and the v heads, in one
    launch.  Caches are [NB, BS, Hk, D] bf16 (store_kvcache) or float8_e4m3fn (the FP8 store,
    per-head scales optional); slot -1 skips a token.  With an FP8 store, k_mirror / v_mirror
    (bf16 caches of the same shape) receive the bf16 rows in the same launch."""
    _cuda(qkv, q_weight, k_weight, cos_sin, positions, k_cache, v_cache, slot_mapping, k_scale, v_scale, k_mirror,
          v_mirror)
    assert qkv.stride(1) == 1 and cos_sin.dtype == torch.float32 and cos_sin.is_contiguous()
    assert positions.dtype == torch.int64 and positions.is_contiguous()
    assert slot_mapping.dtype == torch.int32 and slot_mapping.is_contiguous() and slot_mapping.numel() >= qkv.shape[0]
    assert k_cache.is_contiguous() and v_cache.is_contiguous() and k_cache.shape == v_cache.shape
    assert k_cache.dtype == v_cache.dtype and k_cache.shape[-2:] == (num_kv_heads, head_dim)
    if k_cache.dtype == torch.bfloat16:
        kv_dtype = 0
    else:
        assert k_cache.dtype == torch.float8_e4m3fn
        kv_dtype = 1
    for sc in (k_scale, v_scale):
        assert sc is None or (sc.dtype == torch.float32 and sc.is_contiguous() and sc.numel() == num_kv_heads)
    num_slots = k_cache.numel() // (num_kv_heads * head_dim)
    lib = _lib.load()
    if k_mirror is None and v_mirror is None:
        check(lib.hl_qk_norm_rope_store(qkv.data_ptr(), qkv.stride(0), qkv.shape[0], num_q_heads, num_kv_heads,
                                        head_dim, q_weight.data_ptr(), k_weight.data_ptr(), cos_sin.data_ptr(),
                                        positions.data_ptr(), float(eps), k_cache.data_ptr(), v_cache.data_ptr(),
                                        kv_dtype, slot_mapping.data_ptr(), num_slots, _p(k_scale), _p(v_scale),
                                        _stream(qkv)), "hl_qk_norm_rope_store")
        return
    assert kv_dtype == 1 and k_mirror is not None and v_mirror is not None
    for m in (k_mirror, v_mirror):
        assert m.dtype == torch.bfloat16 and m.is_contiguous() and m.shape == k_cache.shape
    check(lib.hl_qk_norm_rope_store_mirrored(qkv.data_ptr(), qkv.stride(0), qkv.shape[0], num_q_heads, num_kv_heads,
                                             head_dim, q_weight.data_ptr(), k_weight.data_ptr(), cos_sin.data_ptr(),
                                             positions.data_ptr(), float(eps), k_cache.data_ptr(), v_cache.data_ptr(),
                                             kv_dtype, slot_mapping.data_ptr(), num_slots, _p(k_scale), _p(v_scale),
                                             k_mirror.data_ptr(), v_mirror.data_ptr(), _stream(qkv)),
          "hl_qk_norm_rope_store_mirrored")


def sample(logits: torch.Tensor, temperatures: torch.Tensor | None, seed: int, step_state: torch.Tensor | None,
           out: torch.Tensor | None = None, index_offset: int = 0,
           out_values: torch.Tensor | None = None) -> torch.Tensor:
    """Per row: Gumbel-max temperature sample (temperatures[row] > 0) or greedy argmax of bf16
    logits [rows, V] (hl_sample).  step_state: int64 [2] device counter advanced per launch."""
    _cuda(logits, temperatures, step_state, out, out_values)
    rows, vocab = logits.shape
    assert logits.dtype == torch.bfloat16 and logits.stride(1) == 1
    if temperatures is not None:
        assert temperatures.dtype == torch.float32 and temperatures.is_contiguous() and temperatures.numel() >= rows
    if step_state is not None:
        assert step_state.dtype == torch.int64 and step_state.numel() >= 2
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    lib = _lib.load()
    check(lib.hl_sample(logits.data_ptr(), logits.stride(0), rows, vocab, int(index_offset), _p(temperatures),
                        int(seed) & 0xFFFFFFFFFFFFFFFF, _p(step_state), out.data_ptr(), _p(out_values),
                        _stream(logits)), "hl_sample")
    return out


def sample_filtered(logits: torch.Tensor, temperatures: torch.Tensor | None, top_ks: torch.Tensor | None,
                    top_ps: torch.Tensor | None, seed: int, step_state: torch.Tensor | None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """hl_sample with the reference's top-k / top-p filters (mini_vllm/layers/sampler.py:13-49):
    per row a Gumbel-max draw from softmax(logits / T) restricted to the top-k, then top-p, set
    (top_ks int32, <= 0 or >= V: no filter; top_ps float32, >= 1: no filter); greedy argmax where
    T <= 0.  Rows without filters get exactly sample()'s token for the same seed and step."""
    _cuda(logits, temperatures, top_ks, top_ps, step_state, out)
    rows, vocab = logits.shape
    assert logits.dtype == torch.bfloat16 and logits.stride(1) == 1
    for t, dt in ((temperatures, torch.float32), (top_ks, torch.int32), (top_ps, torch.float32)):
        if t is not None:
            assert t.dtype == dt and t.is_contiguous() and t.numel() >= rows
    if step_state is not None:
        assert step_state.dtype == torch.int64 and step_state.numel() >= 2
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    lib = _lib.load()
    check(lib.hl_sample_filtered(logits.data_ptr(), logits.stride(0), rows, vocab, _p(temperatures), _p(top_ks),
                                 _p(top_ps), int(seed) & 0xFFFFFFFFFFFFFFFF, _p(step_state), out.data_ptr(),
                                 _stream(logits)), "hl_sample_filtered")
    return out


def silu_mul(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _cuda(x, out)
    rows, two_i = x.shape
    inter = two_i // 2
    assert x.stride(1) == 1
    if out is None:
        out = torch.empty(rows, inter, dtype=x.dtype, device=x.device)
    lib = _lib.load()
    check(lib.hl_silu_mul(x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0), rows, inter, _stream(x)),
          "hl_silu_mul")
    return out


def argmax(logits: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _cuda(logits, out)
    rows, vocab = logits.shape
    assert logits.dtype == torch.bfloat16 and logits.stride(1) == 1
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    lib = _lib.load()
    check(lib.hl_argmax(logits.data_ptr(), logits.stride(0), rows, vocab, out.data_ptr(), _stream(logits)),
          "hl_argmax")
    return out


def argmax_shard(logits: torch.Tensor, index_offset: int, out_tokens: torch.Tensor, out_values: torch.Tensor):
    """Per-row (max value, index + index_offset) of one vocabulary shard (hl_argmax_shard)."""
    _cuda(logits, out_tokens, out_values)
    rows, vocab = logits.shape
    assert logits.dtype == torch.bfloat16 and logits.stride(1) == 1
    assert out_tokens.dtype == torch.int64 and out_values.dtype == torch.float32
    lib = _lib.load()
    check(lib.hl_argmax_shard(logits.data_ptr(), logits.stride(0), rows, vocab, int(index_offset),
                              out_tokens.data_ptr(), out_values.data_ptr(), _stream(logits)), "hl_argmax_shard")


# ------------------------------------------------------------------------ page tables
# The checks of the operators below are written to be cheap (one stride() or shape per tensor): their
# small calls take less time on the GPU than on the host.
_BF16, _F32, _E4M3, _I32, _I64 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int32, torch.int64


def _on_one_device(first: torch.Tensor, *rest: torch.Tensor) -> None:
    """All tensors (None allowed) on one CUDA device."""
    dev = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != dev:
            _cuda(first, *rest)
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
    if dev < 0:
        _cuda(first)


def _launch(name: str, t: torch.Tensor, *args) -> None:
    """Calls the C entry point `name` on t's device, current or not, and that device's stream."""
    fn = getattr(_lib.load(), name)
    dev = t.get_device()
    if dev == torch._C._cuda_getDevice():
        check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)), name)
    else:
        with torch.cuda.device(dev):
            check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)), name)


def extend_block_tables(block_tables: torch.Tensor, cached_lens: torch.Tensor | None, query_lens: torch.Tensor,
                        free_blocks: torch.Tensor, block_size: int, max_tokens: int) -> dict:
    """Gives every sequence the pages its new tokens need and builds the batch description on the
    device (hl_extend_block_tables): prefill_metadata without the host loop, for lengths and a free
    list that are on the GPU.

    block_tables [B, MB] int32, updated in place: row b keeps its ceil(cached_lens[b] / block_size)
    first entries, takes the next ids of free_blocks [F] int32 for the others it needs, -1 behind
    them.  cached_lens / query_lens [B] int32 (cached_lens None: all 0).  Returns the keys of
    prefill_metadata (block_tables, cu_seqlens_q, cu_seqlens_k, positions int64 and slot_mapping of
    max_tokens entries, 0 / -1 behind the batch's last token) plus context_lens and status, int32
    [2]: pages taken, error bits (1: free list too short, 2: table too narrow, 4: more than
    max_tokens tokens; what did not fit is -1)."""
    _on_one_device(block_tables, query_lens, free_blocks, cached_lens)
    b, width = block_tables.shape
    row, one = block_tables.stride()
    assert block_tables.dtype == _I32 and one == 1
    assert query_lens.dtype == _I32 and query_lens.is_contiguous() and query_lens.shape == (b,)
    assert cached_lens is None or (cached_lens.dtype == _I32 and cached_lens.is_contiguous()
                                   and cached_lens.shape == (b,))
    assert free_blocks.dtype == _I32 and free_blocks.is_contiguous() and free_blocks.dim() == 1
    # One allocation for the int32 results (slots first: 16-byte stores), one for the positions.
    results = query_lens.new_empty(max_tokens + 3 * b + 4)
    slots, cu_q, cu_k, context, status = torch.unsafe_split_with_sizes(results, (max_tokens, b + 1, b + 1, b, 2))
    positions = query_lens.new_empty(max_tokens, dtype=_I64)
    at = results.data_ptr()
    cu_at = at + 4 * max_tokens
    _launch(
        "hl_extend_block_tables", block_tables, None if cached_lens is None else cached_lens.data_ptr(),
        query_lens.data_ptr(), b, block_tables.data_ptr(), row, width, free_blocks.data_ptr(), free_blocks.numel(),
        block_size, max_tokens, cu_at, cu_at + 4 * b + 4, cu_at + 8 * b + 8, positions.data_ptr(), at,
        cu_at + 12 * b + 8)
    return {"block_tables": block_tables, "cu_seqlens_q": cu_q, "cu_seqlens_k": cu_k, "context_lens": context,
            "positions": positions, "slot_mapping": slots, "status": status}


# ------------------------------------------------------------------------ block-scaled 8-bit cache
def _check_block_cache(k_cache, v_cache, k_scales, v_scales):
    """(num_blocks, block_size, Hk, D, scale_block) of a block-scaled cache."""
    shape, scales = k_cache.shape, k_scales.shape
    nb, bs, hk, d = shape
    snb, groups, shk = scales
    assert k_cache.dtype == _E4M3 == v_cache.dtype and v_cache.shape == shape
    assert k_scales.dtype == _F32 == v_scales.dtype and v_scales.shape == scales
    assert (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scales.is_contiguous()
            and v_scales.is_contiguous())
    assert snb == nb and shk == hk and groups > 0 and bs % groups == 0
    return nb, bs, hk, d, bs // groups


def store_kvcache_fp8_blocks(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                             k_scales: torch.Tensor, v_scales: torch.Tensor, block_tables: torch.Tensor,
                             context_lens: torch.Tensor, cu_seqlens_q: torch.Tensor | None = None) -> None:
    """Stores new tokens into an 8-bit cache whose scales follow the data: one power of two per block
    of tokens and head (hl_store_kv_fp8_blocks).

    key/value [N, Hk, D] bf16 (row-strided views allowed); caches [NB, BS, Hk, D] e4m3; scales
    [NB, BS / T, Hk] fp32, T a multiple of 64; block_tables [B, MB] int32; context_lens [B] int32
    including the new tokens; cu_seqlens_q [B + 1] int32, the rows of each sequence (None: one row
    per sequence).  Tokens that a block held before are rescaled when its scale grows; whatever a
    page held for an earlier owner does not count."""
    _on_one_device(key, value, k_cache, v_cache, k_scales, v_scales, block_tables, context_lens, cu_seqlens_q)
    shape = key.shape
    n, hk, hd = shape
    nb, bs, hk2, hd2, t = _check_block_cache(k_cache, v_cache, k_scales, v_scales)
    assert value.shape == shape and hk == hk2 and hd == hd2
    assert key.dtype == _BF16 == value.dtype
    krs, khs, kes = key.stride()
    vrs, vhs, ves = value.stride()
    assert n == 0 or (kes == 1 == ves and khs == hd == vhs)
    rows, width = block_tables.shape
    row, one = block_tables.stride()
    b = context_lens.numel()
    assert block_tables.dtype == _I32 and one == 1 and rows >= b
    assert context_lens.dtype == _I32 and context_lens.is_contiguous()
    cu = None
    if cu_seqlens_q is not None:
        assert cu_seqlens_q.dtype == _I32 and cu_seqlens_q.is_contiguous() and cu_seqlens_q.numel() == b + 1
        cu = cu_seqlens_q.data_ptr()
    if n <= 1:  # a single row may come with any row stride
        krs = vrs = hk * hd
    _launch(
        "hl_store_kv_fp8_blocks", key, key.data_ptr(), value.data_ptr(), krs, vrs, n, k_cache.data_ptr(),
        v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), block_tables.data_ptr(), row, width,
        context_lens.data_ptr(), cu, b, hk, hd, bs, t, nb)


def make_block_decode_workspace(batch: int, num_q_heads: int, num_kv_heads: int, device) -> torch.Tensor:
    """Zero-filled workspace for paged_decode_fp8_blocks; serves every batch up to `batch`."""
    n = _lib.load().hl_paged_decode_fp8_blocks_workspace_size(batch, num_q_heads, num_kv_heads)
    if n < 0:
        raise ValueError("bad decode workspace shape")
    return torch.zeros(n, dtype=torch.uint8, device=device)


def paged_decode_fp8_blocks(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor,
                            v_scales: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                            softmax_scale: float, out: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode over the cache of store_kvcache_fp8_blocks: one new token per sequence, q
    [B, Hq, D] (or [B, 1, Hq, D]) bf16, Hq / Hk <= 16; block_tables [>= B, MB] int32, context_lens
    [>= B] int32.  Returns out [B, Hq, D].  workspace (None: made and zero-filled by every call) from
    make_block_decode_workspace.  Error bits: decode_errors(workspace)."""
    if q.dim() == 4:
        assert q.shape[1] == 1
        q = q.squeeze(1)
    _on_one_device(q, k_cache, v_cache, k_scales, v_scales, block_tables, context_lens, out, workspace)
    shape = q.shape
    b, hq, hd = shape
    nb, bs, hk, hd2, t = _check_block_cache(k_cache, v_cache, k_scales, v_scales)
    qrs, qhs, qes = q.stride()
    assert q.dtype == _BF16 and hd == hd2 and (b == 0 or (qes == 1 and qhs == hd))
    rows, width = block_tables.shape
    row, one = block_tables.stride()
    assert block_tables.dtype == _I32 and one == 1 and rows >= b
    assert context_lens.dtype == _I32 and context_lens.is_contiguous() and context_lens.numel() >= b
    ors = hq * hd
    if out is None:
        out = q.new_empty(b, hq, hd)
    else:
        ors, ohs, oes = out.stride()
        assert out.dtype == _BF16 and out.shape == shape and (b == 0 or (oes == 1 and ohs == hd))
    if b == 0:
        return out
    if workspace is None:
        workspace = make_block_decode_workspace(b, hq, hk, q.device)
    assert workspace.dtype == torch.uint8 and workspace.is_contiguous()
    if b == 1:  # a single row may come with any row stride
        qrs = ors = hq * hd
    _launch(
        "hl_paged_decode_fp8_blocks", q, q.data_ptr(), qrs, k_cache.data_ptr(), v_cache.data_ptr(),
        k_scales.data_ptr(), v_scales.data_ptr(), block_tables.data_ptr(), row, width, context_lens.data_ptr(), b, hq,
        hk, hd, bs, t, nb, softmax_scale, out.data_ptr(), ors, workspace.data_ptr(), workspace.numel())
    return out


# ------------------------------------------------------------------------ log probabilities
def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, top_n: int = 0):
    """Per row of logits [rows, V] (bf16 or fp32): the log probability of token_ids[row] (int64; -inf
    outside the vocabulary), the entropy of the row's distribution and its top_n <= 32 most probable
    tokens, lowest id first among equals (hl_token_logprobs).  Returns (logprobs [rows], entropies
    [rows], top_tokens [rows, top_n] int64, top_logprobs [rows, top_n]), fp32."""
    _on_one_device(logits, token_ids)
    rows, vocab = logits.shape
    row, one = logits.stride()
    dtype = logits.dtype
    assert (dtype == _BF16 or dtype == _F32) and (one == 1 or vocab == 1)
    assert token_ids.dtype == _I64 and token_ids.is_contiguous() and token_ids.shape == (rows,)
    assert 0 <= top_n <= 32 and top_n <= vocab
    logprobs = logits.new_empty(rows, dtype=_F32)
    entropies = logits.new_empty(rows, dtype=_F32)
    top_tokens = token_ids.new_empty(rows, top_n)
    top_logprobs = logits.new_empty(rows, top_n, dtype=_F32)
    _launch(
        "hl_token_logprobs", logits, logits.data_ptr(), 1 if dtype == _F32 else 0, row if rows > 1 else vocab, rows,
        vocab, token_ids.data_ptr(), top_n, logprobs.data_ptr(), entropies.data_ptr(), top_tokens.data_ptr(),
        top_logprobs.data_ptr())
    return logprobs, entropies, top_tokens, top_logprobs
