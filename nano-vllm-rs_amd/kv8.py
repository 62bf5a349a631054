"""The 8-bit KV cache over torch device tensors: quantised write, producer, read-back, attention.

A cache is four tensors: codes [num_blocks, block_size, Hkv, D] in torch.int8 or torch.float8_e4m3fn
(the dtype names the format) and scales f32 [num_blocks, Hkv], K and V apart; `LayerKVCache` makes them
for a `KVCacheConfig` of one of these dtypes.  include/nvllm_attn.h says what a write does to a block.
Activations are bfloat16 or float32.  As in `attention`, tensors are contiguous and on a HIP device, all
of a call on one; a call runs on that device's current stream.
"""
import contextlib

import torch

from . import capi
from .core import KV8_FORMATS, ConfigError, check

_DT = {torch.bfloat16: 0, torch.float32: 1}


def _refuse(message, code=capi.NVLLM_ERR_CONFIG):
    raise ConfigError(code, message)


def _launch(device, *tensors):
    """Checks what every tensor of a call has to be; returns the stream to launch on and the guard to
    launch under."""
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("nano_vllm_rs_amd operators need HIP device tensors (no CPU fallback exists)")
        if t.device != device:
            _refuse("tensors are on different devices: %s and %s" % (device, t.device))
        if not t.is_contiguous():
            _refuse("tensor must be contiguous")
    guard = (contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device))
    return torch.cuda.current_stream(device).cuda_stream, guard


def _cache(key_cache, value_cache, key_scales, value_scales):
    """-> (num_blocks, block_size, Hkv, D, format)"""
    if key_cache.dtype not in KV8_FORMATS:
        _refuse("cache dtype must be int8 or float8_e4m3fn, not %s" % key_cache.dtype, capi.NVLLM_ERR_UNSUPPORTED)
    if key_cache.dim() != 4 or value_cache.shape != key_cache.shape or value_cache.dtype != key_cache.dtype:
        _refuse("key and value cache must be [num_blocks, block_size, Hkv, D] of one dtype")
    nb, bs, hkv, d = key_cache.shape
    for s in (key_scales, value_scales):
        if s.dtype != torch.float32 or s.shape != (nb, hkv):
            _refuse("scales must be float32 [num_blocks, Hkv]")
    return nb, bs, hkv, d, KV8_FORMATS[key_cache.dtype]


def _dtype(t, *same):
    if t.dtype not in _DT:
        _refuse("dtype must be bfloat16 or float32", capi.NVLLM_ERR_UNSUPPORTED)
    for x in same:
        if x is not None and x.dtype != t.dtype:
            _refuse("dtypes differ: %s and %s" % (t.dtype, x.dtype))
    return _DT[t.dtype]


def _write_workspace(workspace, n, bs, nb, device):
    if workspace is None:
        need = capi.lib().nvllm_kv8_write_workspace_bytes(n, bs, nb)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
    return workspace


def _p(t):
    return t.data_ptr() if t is not None else None


def _size(t):
    return t.numel() * t.element_size() if t is not None else 0


def reshape_and_cache_kv8(key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping,
                          workspace=None):
    """nvllm_reshape_and_cache_kv8: key / value [num_tokens, Hkv, D] into the slots of slot_mapping
    (int64 [num_tokens] on the device); updates caches and scales in place.  `workspace`: uint8, of
    nvllm_kv8_write_workspace_bytes; made for the call if None."""
    nb, bs, hkv, d, fmt = _cache(key_cache, value_cache, key_scales, value_scales)
    n = key.shape[0]
    if key.shape != (n, hkv, d) or value.shape != key.shape:
        _refuse("key and value must be [num_tokens, Hkv, D] of the cache")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (n,):
        _refuse("slot_mapping must be int64 [num_tokens]")
    dt = _dtype(key, value)
    dev = key.device
    stream, guard = _launch(dev, key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping, workspace)
    with guard:
        ws = _write_workspace(workspace, n, bs, nb, dev)
        check(capi.lib().nvllm_reshape_and_cache_kv8(
            key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(),
            value_scales.data_ptr(), slot_mapping.data_ptr(), _p(ws), _size(ws), n, hkv, d, bs, nb, fmt, dt, stream))


def qk_norm_rope_cache_kv8(query, key, value, q_weight, k_weight, eps, rotary, positions, key_cache, value_cache,
                           key_scales, value_scales, slot_mapping, k_out=None, q_out=None, workspace=None):
    """nvllm_qk_norm_rope_cache_kv8: `qk_norm_rope_cache` with the rotated K and V going into the 8-bit
    cache.  k_out must not be key.  Returns q_out (query itself unless q_out is given)."""
    nb, bs, hkv, d, fmt = _cache(key_cache, value_cache, key_scales, value_scales)
    n, hq = query.shape[0], query.shape[1]
    if query.shape != (n, hq, d) or key.shape != (n, hkv, d) or value.shape != key.shape:
        _refuse("query must be [num_tokens, Hq, D], key and value [num_tokens, Hkv, D] of the cache")
    if q_weight.shape != (d,) or k_weight.shape != (d,):
        _refuse("q_weight and k_weight must be [D]")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (n,):
        _refuse("slot_mapping must be int64 [num_tokens]")
    if positions.dtype != torch.int32 or positions.shape != (n,):
        _refuse("positions must be int32 [num_tokens]")
    if q_out is None:
        q_out = query
    cos, sin = rotary.cos_cache(), rotary.sin_cache()
    if cos.dim() != 2 or cos.shape[1] != d or sin.shape != cos.shape:
        _refuse("rotary tables must be [positions, D]")
    if q_out.shape != query.shape or (k_out is not None and k_out.shape != key.shape):
        _refuse("q_out / k_out must have the shape of query / key")
    dt = _dtype(query, key, value, q_weight, k_weight, cos, sin, q_out, k_out)
    dev = query.device
    stream, guard = _launch(dev, query, key, value, q_weight, k_weight, cos, sin, positions, key_cache, value_cache,
                            key_scales, value_scales, slot_mapping, k_out, q_out, workspace)
    with guard:
        ws = _write_workspace(workspace, n, bs, nb, dev)
        check(capi.lib().nvllm_qk_norm_rope_cache_kv8(
            query.data_ptr(), key.data_ptr(), value.data_ptr(), q_out.data_ptr(), _p(k_out), q_weight.data_ptr(),
            k_weight.data_ptr(), float(eps), cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(),
            key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
            slot_mapping.data_ptr(), _p(ws), _size(ws), n, hq, hkv, d, bs, nb, fmt, dt, stream))
    return q_out


def gather_cache_blocks_kv8(key_cache, value_cache, key_scales, value_scales, block_ids, dtype=torch.bfloat16):
    """nvllm_gather_cache_blocks_kv8: the values of whole blocks, block_ids int32 [n] on the device ->
    (keys, values), each [n, block_size, Hkv, D] in dtype (exact in either)."""
    nb, bs, hkv, d, fmt = _cache(key_cache, value_cache, key_scales, value_scales)
    if block_ids.dtype != torch.int32 or block_ids.dim() != 1:
        _refuse("block_ids must be int32 [n]")
    if dtype not in _DT:
        _refuse("dtype must be bfloat16 or float32", capi.NVLLM_ERR_UNSUPPORTED)
    dev = key_cache.device
    stream, guard = _launch(dev, key_cache, value_cache, key_scales, value_scales, block_ids)
    n = block_ids.shape[0]
    with guard:
        out = torch.empty((2, n, bs, hkv, d), dtype=dtype, device=dev)
        keys, values = out.unbind(0)
        check(capi.lib().nvllm_gather_cache_blocks_kv8(
            key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
            block_ids.data_ptr(), n, keys.data_ptr(), values.data_ptr(), nb, bs, hkv, d, fmt, _DT[dtype], stream))
    return keys, values


PAGED_KV8_PATHS = ("decode", "tile", "generic")


def paged_attention_kv8_path(num_seqs, num_new_tokens, num_heads, num_kv_heads, head_dim, block_size,
                             max_blocks_per_seq, dtype=torch.bfloat16):
    """nvllm_paged_attn_kv8_path: which kernel a launch of this shape runs (pure query)."""
    code = capi.lib().nvllm_paged_attn_kv8_path(num_seqs, num_new_tokens, num_heads, num_kv_heads, head_dim,
                                                block_size, max_blocks_per_seq, _DT[dtype])
    check(min(code, 0))
    return PAGED_KV8_PATHS[code]


def paged_attention_kv8(query, key_cache, value_cache, key_scales, value_scales, block_tables, context_lens, scale,
                        workspace=None):
    """nvllm_paged_attn_kv8, as `paged_attention_batched`: query [num_seqs, T, Hq, D], block_tables int32
    [num_seqs, max_blocks], context_lens int32 [num_seqs] -> [num_seqs, T, Hq*D].  `workspace`: uint8, of
    nvllm_paged_attn_kv8_workspace_bytes; made for the call if None."""
    nb, bs, hkv, d, fmt = _cache(key_cache, value_cache, key_scales, value_scales)
    if query.dim() != 4 or query.shape[3] != d:
        _refuse("query must be [num_seqs, T, Hq, D] of the cache")
    n, t, hq, _ = query.shape
    if block_tables.dtype != torch.int32 or context_lens.dtype != torch.int32:
        _refuse("block_tables and context_lens must be int32")
    if block_tables.dim() != 2 or block_tables.shape[0] != n or context_lens.shape != (n,):
        _refuse("block_tables must be [num_seqs, max_blocks], context_lens [num_seqs]")
    dt = _dtype(query)
    dev = query.device
    stream, guard = _launch(dev, query, key_cache, value_cache, key_scales, value_scales, block_tables, context_lens,
                            workspace)
    width = block_tables.shape[1]
    L = capi.lib()
    with guard:
        out = torch.empty((n, t, hq * d), dtype=query.dtype, device=dev)
        if workspace is None:
            need = L.nvllm_paged_attn_kv8_workspace_bytes(n, t, hq, hkv, d, bs, width, dt)
            if need:
                workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        check(L.nvllm_paged_attn_kv8(
            query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(),
            value_scales.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), out.data_ptr(), _p(workspace),
            _size(workspace), n, t, hq, hkv, d, bs, width, nb, float(scale), fmt, dt, stream))
    return out
