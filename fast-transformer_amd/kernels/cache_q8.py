"""The KV cache held in 8 bits: its write (head norms, RoPE, quantisation) and the decode attention that reads it.

Codes ``keys`` / ``values`` [B, Hkv, C, D] in ``torch.float8_e4m3fn`` or ``torch.int8`` and FP32 scales
[B, Hkv, ceil(C / block)]: slot t's value is ``code * scale[t // block]``, one scale per block of slots, row and KV
head. ``new_cache_q8`` allocates one. ``qk_rope_cache_q8`` stands where ``qk_rope.qk_rope_cache`` does and
``decode_attention_q8`` where ``decode_attention.decode_attention`` does.

The writer's scales are powers of two (csrc/ftk_rope_q8.hip says why); the attention takes any positive ones. A
cache grows at its end: a write keeps the values of the slots before it in its block (re-scaled in place when the
block's scale must grow) and gives up what came after it there. No counterpart in the reference, whose cache is BF16.
"""

import functools

import torch

from kernels import _native

_calls = _native.calls
#: Slots that may share a scale, and query heads per KV head the attention takes.
BLOCKS = (16, 32, 64, 128)
MAX_GROUP = 16
TYPES = {torch.float8_e4m3fn: _native.Q8_E4M3, torch.int8: _native.Q8_INT8}


def new_cache_q8(batch, kv_heads, capacity, dim, block=64, dtype=torch.float8_e4m3fn, device="cuda"):
    """(keys, values, k_scales, v_scales) of an empty cache: zero codes, scales of 1."""
    if dtype not in TYPES:
        raise ValueError(f"cache type {dtype}: float8_e4m3fn or int8")
    if block not in BLOCKS:
        raise ValueError(f"block {block}: {BLOCKS}")
    shape = (batch, kv_heads, capacity, dim)
    keys, values = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    scales = (torch.ones((batch, kv_heads, -(-capacity // block)), device=device) for _ in range(2))
    return (keys, values, *scales)


@functools.lru_cache(maxsize=None)
def block_of(capacity, blocks):
    """Slots per scale of a cache of ``capacity`` slots with ``blocks`` scales: the only size in BLOCKS that gives so
    many (with one block, whichever holds the cache)."""
    for block in BLOCKS:
        if -(-capacity // block) == blocks:
            return block
    raise ValueError(f"{blocks} scales for {capacity} slots: blocks of 16, 32, 64 or 128 slots")


def _check(keys, values, k_scales, v_scales):
    """The cache's checks; returns (type, block)."""
    if keys.dtype not in TYPES or values.dtype != keys.dtype or k_scales.dtype != torch.float32 or \
            v_scales.dtype != torch.float32:
        raise ValueError(f"an 8-bit cache has float8_e4m3fn or int8 codes and FP32 scales, got {keys.dtype}, "
                         f"{values.dtype}, {k_scales.dtype}, {v_scales.dtype}")
    shape = keys.shape
    if values.shape != shape or k_scales.shape[:2] != shape[:2] or k_scales.shape != v_scales.shape or \
            k_scales.dim() != 3:
        raise ValueError(f"keys {tuple(shape)}, values {tuple(values.shape)}, scales {tuple(k_scales.shape)}, "
                         f"{tuple(v_scales.shape)} do not fit together")
    if shape[3] not in (64, 128):
        raise ValueError(f"head_dim {shape[3]}: these kernels take 64 or 128")
    if not (keys.is_contiguous() and values.is_contiguous() and k_scales.is_contiguous() and v_scales.is_contiguous()):
        raise ValueError("the cache's codes and scales must be contiguous")
    if (keys.data_ptr() | values.data_ptr()) & 15:
        raise ValueError("the cache's codes must be 16-byte aligned")
    return TYPES[keys.dtype], block_of(shape[2], k_scales.shape[2])


def _one_device(*tensors):
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on {tensors[0].device} and {t.device}")
    _native.require_gpu(tensors[0])


def qk_rope_cache_q8(packed, q_norm, k_norm, cos, sin, position, keys, values, k_scales, v_scales, q_heads,
                     prefill=False, rows=False, phases=None):
    """``qk_rope_cache`` into an 8-bit cache: the same arguments and result ([B, Hq, T, D], a view of token-major
    storage), FP32 from the packed BF16 QKV [B, T, (Hq + 2 Hkv) D] to one rounding of each query (BF16), key and value
    (a code). Slots outside the cache, and tokens whose phase lies outside the tables, are skipped."""
    query = _calls.write(packed, q_norm.weight, k_norm.weight, q_norm.variance_epsilon, k_norm.variance_epsilon, cos, sin,
                         position, keys, values, k_scales, v_scales, q_heads, prefill, rows, phases)
    if query is not None:
        return query
    kind, block = _check(keys, values, k_scales, v_scales)
    batch, kv_heads, capacity, dim = keys.shape
    q_weight, k_weight = q_norm.weight, k_norm.weight
    if packed.dim() != 3 or packed.shape[0] != batch or packed.shape[2] != (q_heads + 2 * kv_heads) * dim:
        raise ValueError(f"packed QKV {tuple(packed.shape)} for {batch} rows, {q_heads} + 2 x {kv_heads} heads of {dim}")
    tokens = packed.shape[1]
    if q_heads < 1 or kv_heads < 1:
        raise ValueError(f"{q_heads} query and {kv_heads} KV heads: at least one of each")
    for name, t in (("packed", packed), ("cos", cos), ("sin", sin), ("q_norm", q_weight), ("k_norm", k_weight)):
        if t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be BF16, got {t.dtype}")
    if not (packed.is_contiguous() and cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("packed, cos and sin must be contiguous")
    if q_weight.numel() != dim or k_weight.numel() != dim:
        raise ValueError(f"head norms of {q_weight.numel()} and {k_weight.numel()} gains for heads of {dim}")
    if tokens > capacity:
        raise ValueError(f"{tokens} tokens for {capacity} slots")
    if rows and prefill:
        raise ValueError("a prompt fills every row from slot 0: rows has no meaning there")
    if phases is not None:
        if not rows or phases.shape != (batch, tokens) or not phases.is_contiguous() or phases.dtype != torch.int64:
            raise ValueError(f"phases (with rows) must be contiguous int64 [{batch}, {tokens}]")
        if cos.shape != sin.shape or cos.shape[-1] != dim:
            raise ValueError("cos and sin must be whole [table rows, D] tables")
    elif not cos.numel() == sin.numel() == (batch if rows else 1) * tokens * dim:
        raise ValueError(f"cos and sin must hold {(batch if rows else 1) * tokens} rows of {dim}")
    if position.dtype != torch.int64 or position.shape != ((tokens,) if prefill else (batch,) if rows else (1,)) or \
            not position.is_contiguous():
        raise ValueError(f"position {position.dtype} {tuple(position.shape)} does not fit the call")
    _one_device(packed, keys, values, k_scales, v_scales, cos, sin, position, q_weight, k_weight, phases)
    query = torch.empty((batch, tokens, q_heads, dim), device=packed.device, dtype=torch.bfloat16)
    if query.numel():
        mode = (_native.ROPE_PREFILL if prefill else 0) | (_native.ROPE_ROWS if rows else 0) | \
            (_native.ROPE_TABLE if phases is not None else 0)
        q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
        _native.call_on(packed, "ftk_qk_rope_cache_q8", packed.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(),
                        q_norm.variance_epsilon, k_norm.variance_epsilon, cos.data_ptr(), sin.data_ptr(),
                        cos.numel() // dim, position.data_ptr(), _native.ptr(phases), query.data_ptr(),
                        keys.data_ptr(), values.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), batch, tokens,
                        q_heads, kv_heads, capacity, dim, block, kind, mode)
    return query.transpose(1, 2)


@functools.lru_cache(maxsize=None)
def _launch(device, batch, q_heads, kv_heads, capacity, dim, splits):
    """(intervals, workspace bytes) of a shape on a device."""
    if not 0 <= splits < 1 << 31:
        raise ValueError(f"{splits} intervals")
    if splits == 0:
        with torch.cuda.device(device):
            splits = _native.lib().ftk_decode_attention_q8_splits(batch, q_heads, kv_heads, capacity, dim, 0)
    need = _native.lib().ftk_decode_attention_q8_workspace_bytes(batch, q_heads, kv_heads, dim, max(splits, 1))
    if splits < 1 or need < 0:
        raise ValueError(f"decode attention does not take {batch} x {q_heads} / {kv_heads} heads of {dim}, "
                         f"{capacity} slots, {splits} intervals")
    return splits, need


def decode_attention_q8(query, keys, values, k_scales, v_scales, position, scale, splits=0):
    """Q [B, Hq, 1, D] BF16 over an 8-bit cache -> [B, 1, Hq, D]: each row attends to slots 0..position.

    ``position`` int64 [1] (every row's) or [B], on the device; a row whose position is below 0 gives zeros, and one
    past the cache sees all of it. Slots after the position may hold anything. FP32 scores and sums; p weights V as
    two BF16 values that carry 16 bits of it. ``splits``: slot intervals per KV head (0: the planner's).
    """
    out = _calls.attend(query, keys, values, k_scales, v_scales, position, scale, splits)
    if out is not None:
        return out
    kind, block = _check(keys, values, k_scales, v_scales)
    batch, kv_heads, capacity, dim = keys.shape
    if query.dtype != torch.bfloat16 or query.dim() != 4 or query.shape[0] != batch or query.shape[2] != 1 or \
            query.shape[3] != dim:
        raise ValueError(f"query must be BF16 [{batch}, heads, 1, {dim}], got {query.dtype} {tuple(query.shape)}")
    q_heads = query.shape[1]
    if not kv_heads or not q_heads or q_heads % kv_heads or q_heads // kv_heads > MAX_GROUP:
        raise ValueError(f"{q_heads} query heads for {kv_heads} KV heads: a multiple, at most {MAX_GROUP} to one")
    if position.dtype != torch.int64 or position.dim() != 1 or position.shape[0] not in (1, batch) or \
            not position.is_contiguous():
        raise ValueError(f"position must be contiguous int64 [1] or [{batch}], got {position.dtype} {tuple(position.shape)}")
    _one_device(query, keys, values, k_scales, v_scales, position)
    out = torch.empty((batch, 1, q_heads, dim), device=query.device, dtype=torch.bfloat16)
    if not batch:
        return out
    if not query.is_contiguous() or query.data_ptr() & 15:
        query = query.clone(memory_format=torch.contiguous_format)
    splits, need = _launch(query.get_device(), batch, q_heads, kv_heads, capacity, dim, splits)
    # The partials live in memory of this call's own (a graph's own, when captured): calls on different streams, and
    # graphs replayed side by side, never share them.
    ws = torch.empty(need, device=query.device, dtype=torch.uint8) if need else None
    _native.call_on(query, "ftk_decode_attention_q8", query.data_ptr(), keys.data_ptr(), values.data_ptr(),
                    k_scales.data_ptr(), v_scales.data_ptr(), position.data_ptr(), position.shape[0], out.data_ptr(),
                    batch, q_heads, kv_heads, capacity, dim, block, kind, scale, splits, _native.ptr(ws), need)
    return out
