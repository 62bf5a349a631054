"""The 8-bit KV cache over torch device tensors: quantised write, producer, read-back, attention.

A cache is four tensors: codes [num_blocks, block_size, Hkv, D] in torch.int8 or torch.float8_e4m3fn
(the dtype names the format) and scales f32 [num_blocks, Hkv], K and V apart; `LayerKVCache` makes them
for a `KVCacheConfig` of one of these dtypes.  include/nvllm_attn.h says what a write does to a block.
Activations are bfloat16 or float32.  As in `attention`, tensors are contiguous and on a HIP device, all
of a call on one; a call runs on that device's current stream.
"""
import torch

from . import capi
from .core import ConfigError, check

_DT = {torch.bfloat16: 0, torch.float32: 1}
_FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}


def _refuse(message, code=capi.NVLLM_ERR_CONFIG):
    raise ConfigError(code, message)


# the current stream's handle and device (the public ways make a Stream object and look for an initialised
# runtime each time, 2 us of a call's 10)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(tensors):
    """Checks what every tensor of a call has to be; -> the device index."""
    at = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != at or not t.is_contiguous()):
            break
    else:
        if at >= 0:
            return at
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("nano_vllm_rs_amd operators need HIP device tensors (no CPU fallback exists)")
        if t is not None and t.get_device() != at:
            _refuse("tensors are on different devices: %d and %d" % (at, t.get_device()))
    _refuse("tensor must be contiguous")


def _cache(key_cache, value_cache, key_scales, value_scales):
    """-> (num_blocks, block_size, Hkv, D, format)"""
    fmt = _FORMATS.get(key_cache.dtype)
    if fmt is None:
        _refuse("cache dtype must be int8 or float8_e4m3fn, not %s" % key_cache.dtype, capi.NVLLM_ERR_UNSUPPORTED)
    shape = key_cache.shape
    if len(shape) != 4 or value_cache.shape != shape or value_cache.dtype != key_cache.dtype:
        _refuse("key and value cache must be [num_blocks, block_size, Hkv, D] of one dtype")
    nb, bs, hkv, d = shape
    if (key_scales.dtype != torch.float32 or value_scales.dtype != torch.float32 or
            key_scales.shape != (nb, hkv) or value_scales.shape != (nb, hkv)):
        _refuse("scales must be float32 [num_blocks, Hkv]")
    return nb, bs, hkv, d, fmt


def _dtype(t, *same):
    dtype = t.dtype
    code = _DT.get(dtype)
    if code is None:
        _refuse("dtype must be bfloat16 or float32", capi.NVLLM_ERR_UNSUPPORTED)
    for x in same:
        if x is not None and x.dtype != dtype:
            _refuse("dtypes differ: %s and %s" % (dtype, x.dtype))
    return code


def _write_workspace(workspace, n, bs, nb, like):
    if workspace is None:
        need = capi.lib().nvllm_kv8_write_workspace_bytes(n, bs, nb)
        if not need:
            return None, 0
        workspace = like.new_empty((need,), dtype=torch.uint8)
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _p(t):
    return t.data_ptr() if t is not None else None


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
    index = _launch((key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping, workspace))
    if index != _current_device():
        with torch.cuda.device(index):
            return reshape_and_cache_kv8(key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping,
                                         workspace)
    ws, size = _write_workspace(workspace, n, bs, nb, key)
    check(capi.lib().nvllm_reshape_and_cache_kv8(
        key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(),
        value_scales.data_ptr(), slot_mapping.data_ptr(), ws, size, n, hkv, d, bs, nb, fmt, dt, _raw_stream(index)))


def qk_norm_rope_cache_kv8(query, key, value, q_weight, k_weight, eps, rotary, positions, key_cache, value_cache,
                           key_scales, value_scales, slot_mapping, k_out=None, q_out=None, workspace=None):
    """nvllm_qk_norm_rope_cache_kv8: `qk_norm_rope_cache` with the rotated K and V going into the 8-bit
    cache.  q_out is query or overlaps none of query, key and value; k_out overlaps none of the four.  Returns q_out
    (query itself unless q_out is given)."""
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
    index = _launch((query, key, value, q_weight, k_weight, cos, sin, positions, key_cache, value_cache, key_scales,
                     value_scales, slot_mapping, k_out, q_out, workspace))
    if index != _current_device():
        with torch.cuda.device(index):
            return qk_norm_rope_cache_kv8(query, key, value, q_weight, k_weight, eps, rotary, positions, key_cache,
                                          value_cache, key_scales, value_scales, slot_mapping, k_out, q_out, workspace)
    ws, size = _write_workspace(workspace, n, bs, nb, query)
    check(capi.lib().nvllm_qk_norm_rope_cache_kv8(
        query.data_ptr(), key.data_ptr(), value.data_ptr(), q_out.data_ptr(), _p(k_out), q_weight.data_ptr(),
        k_weight.data_ptr(), float(eps), cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(),
        key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
        slot_mapping.data_ptr(), ws, size, n, hq, hkv, d, bs, nb, fmt, dt, _raw_stream(index)))
    return q_out


def gather_cache_blocks_kv8(key_cache, value_cache, key_scales, value_scales, block_ids, dtype=torch.bfloat16):
    """nvllm_gather_cache_blocks_kv8: the values of whole blocks, block_ids int32 [n] on the device ->
    (keys, values), each [n, block_size, Hkv, D] in dtype (exact, but for values below
    bfloat16's smallest number, 2^-133)."""
    nb, bs, hkv, d, fmt = _cache(key_cache, value_cache, key_scales, value_scales)
    if block_ids.dtype != torch.int32 or block_ids.dim() != 1:
        _refuse("block_ids must be int32 [n]")
    if dtype not in _DT:
        _refuse("dtype must be bfloat16 or float32", capi.NVLLM_ERR_UNSUPPORTED)
    index = _launch((key_cache, value_cache, key_scales, value_scales, block_ids))
    if index != _current_device():
        with torch.cuda.device(index):
            return gather_cache_blocks_kv8(key_cache, value_cache, key_scales, value_scales, block_ids, dtype)
    n = block_ids.shape[0]
    keys = key_cache.new_empty((n, bs, hkv, d), dtype=dtype)
    values = key_cache.new_empty((n, bs, hkv, d), dtype=dtype)
    check(capi.lib().nvllm_gather_cache_blocks_kv8(
        key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
        block_ids.data_ptr(), n, keys.data_ptr(), values.data_ptr(), nb, bs, hkv, d, fmt, _DT[dtype],
        _raw_stream(index)))
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
    shape, table = query.shape, block_tables.shape
    if len(shape) != 4 or shape[3] != d:
        _refuse("query must be [num_seqs, T, Hq, D] of the cache")
    n, t, hq, _ = shape
    if block_tables.dtype != torch.int32 or context_lens.dtype != torch.int32:
        _refuse("block_tables and context_lens must be int32")
    if len(table) != 2 or table[0] != n or context_lens.shape != (n,):
        _refuse("block_tables must be [num_seqs, max_blocks], context_lens [num_seqs]")
    width, dt = table[1], _dtype(query)
    index = _launch((query, key_cache, value_cache, key_scales, value_scales, block_tables, context_lens, workspace))
    if index != _current_device():
        with torch.cuda.device(index):
            return paged_attention_kv8(query, key_cache, value_cache, key_scales, value_scales, block_tables,
                                       context_lens, scale, workspace)
    L = capi.lib()
    out = query.new_empty((n, t, hq * d))
    if workspace is None:
        need = L.nvllm_paged_attn_kv8_workspace_bytes(n, t, hq, hkv, d, bs, width, dt)
        if need:
            workspace = query.new_empty((need,), dtype=torch.uint8)
    size = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(L.nvllm_paged_attn_kv8(
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(),
        value_scales.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), out.data_ptr(), _p(workspace),
        size, n, t, hq, hkv, d, bs, width, nb, float(scale), fmt, dt, _raw_stream(index)))
    return out
