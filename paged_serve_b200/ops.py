"""Tensor-level entry points over the C ABI (one function per exported kernel).

Each function validates shapes/dtypes/devices on the host, extracts raw
pointers and strides, and launches on the tensor's current CUDA stream. None
of them synchronises or allocates except where an ``out=`` buffer is omitted.
There is no fallback path: a CPU tensor or a missing library raises.

KV pool layout (per layer): ``[num_blocks, num_kv_heads, block_size, head_dim]``.
"""

from __future__ import annotations

import math

import torch

from paged_serve_b200 import _lib

__all__ = [
    "build_slot_mapping",
    "cache_append",
    "cache_append_quant",
    "cache_append_rope",
    "cache_append_rope_quant",
    "cache_read_quant",
    "copy_blocks",
    "check_block_pairs",
    "decode_plan",
    "decode_workspace_bytes",
    "paged_decode",
    "paged_decode_listed",
    "paged_decode_quant",
    "paged_decode_shared",
    "paged_prefill",
    "stream_read",
    "swap_blocks",
]

# Code types of an 8-bit cache.
CODES = {torch.float8_e4m3fn: _lib.PS_CODE_E4M3, torch.int8: _lib.PS_CODE_INT8}

_DTYPES = {torch.bfloat16: _lib.PS_DTYPE_BF16, torch.float16: _lib.PS_DTYPE_F16}


def _dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {t.dtype}; the CUDA path runs bf16 or fp16") from None


def _require_cuda(*tensors: torch.Tensor | None) -> torch.device:
    first, index = None, -2
    for t in tensors:
        if t is None:
            continue
        i = t.get_device()  # -1 on the CPU; cheaper than comparing device objects
        if i != index:
            if i < 0:
                raise ValueError("paged_serve_b200 kernels need CUDA tensors (no CPU fallback)")
            if first is not None:
                raise ValueError(f"tensors on different devices: {first.device} vs {t.device}")
            first, index = t, i
    assert first is not None
    return first.device


def _stream(device: torch.device) -> int:
    # The handle of torch.cuda.current_stream(device) without making a Stream object (3.8 us
    # of a call's 8 to 20 us on the host), by the function under that property; torch
    # documents neither that one nor another way to the bare handle.
    return torch._C._cuda_getCurrentRawStream(device.index)


def _launch(device: torch.device, fn, *args) -> int:
    """Calls ``fn`` with ``device`` current (the runtime launches on the current device)."""
    if device.index == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check_pool(pool: torch.Tensor, name: str) -> None:
    if len(pool.shape) != 4 or not pool.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [num_blocks, kv_heads, block_size, head_dim]")


def _check_rows(x: torch.Tensor, name: str, heads: int, head_dim: int) -> int:
    """x is [rows, heads, head_dim] with unit dim stride and head stride head_dim."""
    shape = x.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim:
        raise ValueError(f"{name} must be [rows, {heads}, {head_dim}], got {tuple(shape)}")
    row, head, unit = x.stride()
    if unit != 1 or head != head_dim:
        raise ValueError(f"{name} must have contiguous heads (strides (*, {head_dim}, 1))")
    return row if shape[0] > 1 else heads * head_dim


def _err_ptr(device_error: torch.Tensor | None) -> int | None:
    if device_error is None:
        return None
    if device_error.dtype != torch.int32 or device_error.numel() < 1:
        raise ValueError("device_error must be an int32 tensor with at least one element")
    return device_error.data_ptr()


def cache_append(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    slot_mapping: torch.Tensor,
    device_error: torch.Tensor | None = None,
) -> None:
    """Scatter ``key``/``value`` ([T, Hkv, D]) into the pools at ``slot_mapping`` ([T] int64).

    The KV write of ``ContiguousAttentionBackend.forward``
    (pagedserve/attention/contiguous.py:187-189), addressed through slots.
    """
    dev = _require_cuda(k_pool, v_pool, key, value, slot_mapping, device_error)
    _check_pool(k_pool, "k_pool")
    _check_pool(v_pool, "v_pool")
    nb, hkv, bs, d = k_pool.shape
    if v_pool.shape != k_pool.shape or key.dtype != k_pool.dtype or value.dtype != k_pool.dtype:
        raise ValueError("k_pool/v_pool/key/value must share shape and dtype")
    ks = _check_rows(key, "key", hkv, d)
    vs = _check_rows(value, "value", hkv, d)
    t = key.shape[0]
    if value.shape[0] != t or slot_mapping.shape != (t,) or slot_mapping.dtype != torch.int64:
        raise ValueError("slot_mapping must be int64 [num_tokens] matching key/value")
    if not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous")
    lib = _lib.load()
    st = lib.ps_cache_append(
        k_pool.data_ptr(), v_pool.data_ptr(), key.data_ptr(), value.data_ptr(),
        slot_mapping.data_ptr(), t, ks, vs, hkv, d, bs, nb, _dtype_code(k_pool),
        _err_ptr(device_error), _stream(dev),
    )
    _lib.check(st, "cache_append")


def cache_append_rope(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    slot_mapping: torch.Tensor,
    positions: torch.Tensor,
    cos_sin_table: torch.Tensor,
    device_error: torch.Tensor | None = None,
) -> None:
    """``cache_append`` with split-half RoPE applied to K on the way in.

    ``cos_sin_table`` is ``[max_positions, head_dim]`` in the pool dtype: row p is
    cos(p*inv_freq) then sin(p*inv_freq) (see :func:`paged_serve_b200.rope.cos_sin_table`).
    Bit-identical to the reference's ``apply_rotary`` (pagedserve/model/layers.py:62-77).
    """
    dev = _require_cuda(k_pool, v_pool, key, value, slot_mapping, positions, cos_sin_table,
                        device_error)
    _check_pool(k_pool, "k_pool")
    _check_pool(v_pool, "v_pool")
    nb, hkv, bs, d = k_pool.shape
    if v_pool.shape != k_pool.shape or key.dtype != k_pool.dtype or value.dtype != k_pool.dtype:
        raise ValueError("k_pool/v_pool/key/value must share shape and dtype")
    ks = _check_rows(key, "key", hkv, d)
    vs = _check_rows(value, "value", hkv, d)
    t = key.shape[0]
    if value.shape[0] != t or slot_mapping.shape != (t,) or slot_mapping.dtype != torch.int64:
        raise ValueError("slot_mapping must be int64 [num_tokens] matching key/value")
    if positions.shape != (t,) or positions.dtype != torch.int64:
        raise ValueError("positions must be int64 [num_tokens]")
    if not (slot_mapping.is_contiguous() and positions.is_contiguous()):
        raise ValueError("slot_mapping and positions must be contiguous")
    if (cos_sin_table.dim() != 2 or cos_sin_table.shape[1] != d
            or cos_sin_table.dtype != k_pool.dtype or not cos_sin_table.is_contiguous()):
        raise ValueError(f"cos_sin_table must be contiguous [positions, {d}] of the pool dtype")
    lib = _lib.load()
    st = lib.ps_cache_append_rope(
        k_pool.data_ptr(), v_pool.data_ptr(), key.data_ptr(), value.data_ptr(),
        slot_mapping.data_ptr(), positions.data_ptr(), t, ks, vs, hkv, d, bs, nb,
        cos_sin_table.data_ptr(), cos_sin_table.shape[0], d, _dtype_code(k_pool),
        _err_ptr(device_error), _stream(dev),
    )
    _lib.check(st, "cache_append_rope")


def _check_quant_pools(k_pool, v_pool, k_scale, v_scale) -> int:
    """Checks an 8-bit cache's pools and scales; returns their code type."""
    _check_pool(k_pool, "k_pool")
    _check_pool(v_pool, "v_pool")
    dtype, shape = k_pool.dtype, k_pool.shape
    code = CODES.get(dtype)
    if code is None:
        raise ValueError(f"an 8-bit cache holds float8_e4m3fn or int8 codes, not {dtype}")
    if v_pool.shape != shape or v_pool.dtype != dtype:
        raise ValueError("k_pool/v_pool must share shape and dtype")
    rows = shape[:3]
    for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if t.dtype != torch.float32 or t.shape != rows or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 [num_blocks, kv_heads, block_size]")
    return code


def _append_quant(what, k_pool, v_pool, k_scale, v_scale, key, value, slot_mapping, positions,
                  cos_sin_table, device_error) -> None:
    dev = _require_cuda(k_pool, v_pool, k_scale, v_scale, key, value, slot_mapping, positions,
                        cos_sin_table, device_error)
    code = _check_quant_pools(k_pool, v_pool, k_scale, v_scale)
    nb, hkv, bs, d = k_pool.shape
    if key.dtype != value.dtype:
        raise ValueError("key/value must share a dtype")
    ks = _check_rows(key, "key", hkv, d)
    vs = _check_rows(value, "value", hkv, d)
    t = key.shape[0]
    if value.shape[0] != t or slot_mapping.shape != (t,) or slot_mapping.dtype != torch.int64:
        raise ValueError("slot_mapping must be int64 [num_tokens] matching key/value")
    if not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous")
    pools = (k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
             key.data_ptr(), value.data_ptr(), slot_mapping.data_ptr())
    tail = (_dtype_code(key), code, _err_ptr(device_error), _stream(dev))
    lib = _lib.load()
    if positions is None:
        st = _launch(dev, lib.ps_cache_append_quant, *pools, t, ks, vs, hkv, d, bs, nb, *tail)
    else:
        if positions.shape != (t,) or positions.dtype != torch.int64 or \
                not positions.is_contiguous():
            raise ValueError("positions must be contiguous int64 [num_tokens]")
        table_shape = cos_sin_table.shape
        if (len(table_shape) != 2 or table_shape[1] != d or cos_sin_table.dtype != key.dtype
                or not cos_sin_table.is_contiguous()):
            raise ValueError(f"cos_sin_table must be contiguous [positions, {d}] of the key dtype")
        st = _launch(dev, lib.ps_cache_append_rope_quant, *pools, positions.data_ptr(), t, ks, vs,
                     hkv, d, bs, nb, cos_sin_table.data_ptr(), table_shape[0], d, *tail)
    _lib.check(st, what)


def cache_append_quant(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    slot_mapping: torch.Tensor,
    device_error: torch.Tensor | None = None,
) -> None:
    """:func:`cache_append` into an 8-bit cache: quantises each row as it is written.

    The pools hold codes (``float8_e4m3fn`` or ``int8``), ``k_scale``/``v_scale`` one
    float32 scale per row (``[num_blocks, Hkv, block_size]``). For a row x,
    ``scale = max(max|x| / qmax, 2**-126)`` (qmax 448 or 127) and
    ``code = round(x * (1 / scale))``, each step in float32; the value is
    ``code * scale``. The reference's cache holds the model's dtype and has no counterpart.
    """
    _append_quant("cache_append_quant", k_pool, v_pool, k_scale, v_scale, key, value,
                  slot_mapping, None, None, device_error)


def cache_append_rope_quant(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    slot_mapping: torch.Tensor,
    positions: torch.Tensor,
    cos_sin_table: torch.Tensor,
    device_error: torch.Tensor | None = None,
) -> None:
    """:func:`cache_append_quant` with split-half RoPE applied to K on the way in.

    K is rotated in float32 with ``cos_sin_table`` (:func:`paged_serve_b200.rope.cos_sin_table`,
    in the key's dtype) and quantised from there, without the roundings to the
    storage type that :func:`cache_append_rope` makes.
    """
    if positions is None or cos_sin_table is None:
        raise ValueError("cache_append_rope_quant needs positions and cos_sin_table")
    _append_quant("cache_append_rope_quant", k_pool, v_pool, k_scale, v_scale, key, value,
                  slot_mapping, positions, cos_sin_table, device_error)


def cache_read_quant(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    ctx_lens: torch.Tensor,
    k_out: torch.Tensor,
    v_out: torch.Tensor,
    out_tables: torch.Tensor,
    device_error: torch.Tensor | None = None,
) -> None:
    """Tokens ``[0, ctx_lens[b])`` of each sequence back from an 8-bit cache.

    Block j of sequence b goes from pool block ``block_tables[b, j]`` to block
    ``out_tables[b, j]`` of the bf16/fp16 pools ``k_out``/``v_out`` (same heads, block
    size and head dim, any number of blocks) as ``code * scale``, rounded once; rows
    past the last token become zeros and other blocks stay as they are.
    :func:`paged_prefill` and :func:`paged_decode_shared` run on the result with
    ``out_tables``.
    """
    dev = _require_cuda(k_pool, v_pool, k_scale, v_scale, block_tables, ctx_lens, k_out, v_out,
                        out_tables, device_error)
    code = _check_quant_pools(k_pool, v_pool, k_scale, v_scale)
    _check_pool(k_out, "k_out")
    _check_pool(v_out, "v_out")
    nb, hkv, bs, d = k_pool.shape
    if k_out.shape[1:] != k_pool.shape[1:] or v_out.shape != k_out.shape or \
            v_out.dtype != k_out.dtype:
        raise ValueError("k_out/v_out must share shape and dtype and match the pools' block shape")
    b = ctx_lens.shape[0]
    if ctx_lens.dtype != torch.int32 or ctx_lens.shape != (b,) or not ctx_lens.is_contiguous():
        raise ValueError("ctx_lens must be contiguous int32 [num_seqs]")
    for t, name in ((block_tables, "block_tables"), (out_tables, "out_tables")):
        if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != b or \
                t.shape[1] != block_tables.shape[1]:
            raise ValueError(f"{name} must be int32 [num_seqs, max_blocks]")
        if t.stride(1) != 1:
            raise ValueError(f"{name} rows must be contiguous")
    w = block_tables.shape[1]
    if b == 0 or w == 0:
        return
    st = _launch(
        dev, _lib.load().ps_cache_read_quant, k_pool.data_ptr(), v_pool.data_ptr(),
        k_scale.data_ptr(), v_scale.data_ptr(), nb, k_out.data_ptr(), v_out.data_ptr(),
        k_out.shape[0], block_tables.data_ptr(), block_tables.stride(0) if b > 1 else w,
        out_tables.data_ptr(), out_tables.stride(0) if b > 1 else w, ctx_lens.data_ptr(), b, hkv, d,
        bs, w, _dtype_code(k_out), code, _err_ptr(device_error), _stream(dev),
    )
    _lib.check(st, "cache_read_quant")


def check_block_pairs(pairs) -> None:
    """Raise ValueError unless a copy list is defined for one concurrent launch.

    ``pairs``: (src, dst) rows as a list or an [N, 2] tensor. Every destination
    must be distinct and no destination may be another pair's source; a chain
    such as (a, b), (b, c) has to be split into two calls in order.
    """
    rows = pairs.tolist() if isinstance(pairs, torch.Tensor) else [tuple(p) for p in pairs]
    dsts = [int(d) for _, d in rows]
    seen: set[int] = set()
    for d in dsts:
        if d in seen:
            raise ValueError(f"copy_blocks: destination block {d} appears twice")
        seen.add(d)
    count: dict[int, int] = {}
    for s, _ in rows:
        count[int(s)] = count.get(int(s), 0) + 1
    for s, d in rows:
        if count.get(int(d), 0) - (1 if int(s) == int(d) else 0) > 0:
            raise ValueError(f"copy_blocks: destination block {d} is another pair's source")


def copy_blocks(
    k_pools: torch.Tensor,
    v_pools: torch.Tensor,
    block_pairs: torch.Tensor,
    device_error: torch.Tensor | None = None,
    check: bool = False,
) -> None:
    """``pool[dst] = pool[src]`` for every (src, dst) row of ``block_pairs`` ([N, 2] int64).

    Pools are one layer ``[num_blocks, Hkv, bs, D]`` or all layers
    ``[L, num_blocks, Hkv, bs, D]`` (copied in one launch). All pairs run at
    once, so every destination must be distinct and none may be another
    pair's source (:func:`check_block_pairs`). ``check=True`` verifies that on
    the host first (reads the pairs back: a synchronising debug aid); the
    kernel itself flags violations in lists of up to 4096 pairs with
    ``PS_DEVERR_BLOCK_PAIRS`` in ``device_error``.
    """
    dev = _require_cuda(k_pools, v_pools, block_pairs, device_error)
    if check:
        check_block_pairs(block_pairs.cpu())
    if k_pools.shape != v_pools.shape or k_pools.dtype != v_pools.dtype:
        raise ValueError("k_pools and v_pools must match")
    if k_pools.dim() == 4:
        layers, layer_stride = 1, 0
        nb = k_pools.shape[0]
    elif k_pools.dim() == 5:
        layers = k_pools.shape[0]
        nb = k_pools.shape[1]
        layer_stride = k_pools.stride(0) * k_pools.element_size()
    else:
        raise ValueError("pools must be [blocks, Hkv, bs, D] or [L, blocks, Hkv, bs, D]")
    if not (k_pools.is_contiguous() and v_pools.is_contiguous()):
        raise ValueError("pools must be contiguous")
    if block_pairs.dtype != torch.int64 or block_pairs.dim() != 2 or block_pairs.shape[1] != 2:
        raise ValueError("block_pairs must be int64 [num_pairs, 2]")
    if not block_pairs.is_contiguous():
        raise ValueError("block_pairs must be contiguous")
    block_bytes = math.prod(k_pools.shape[-3:]) * k_pools.element_size()
    lib = _lib.load()
    st = lib.ps_copy_blocks(
        k_pools.data_ptr(), v_pools.data_ptr(), block_pairs.data_ptr(), block_pairs.shape[0],
        layers, layer_stride, block_bytes, nb, _err_ptr(device_error), _stream(dev),
    )
    _lib.check(st, "copy_blocks")


def _pool_geometry(pool: torch.Tensor) -> tuple[int, int, int]:
    """(layers, blocks, layer stride in bytes) of a [blocks, ...] or [L, blocks, ...] pool."""
    if pool.dim() == 4:
        return 1, pool.shape[0], 0
    if pool.dim() == 5:
        return pool.shape[0], pool.shape[1], pool.stride(0) * pool.element_size()
    raise ValueError("pools must be [blocks, Hkv, bs, D] or [L, blocks, Hkv, bs, D]")


def swap_blocks(
    dst_k: torch.Tensor,
    dst_v: torch.Tensor,
    src_k: torch.Tensor,
    src_v: torch.Tensor,
    block_pairs: torch.Tensor,
    max_ctas: int = 0,
    device_error: torch.Tensor | None = None,
    stream: torch.cuda.Stream | None = None,
) -> None:
    """``dst[d] = src[s]`` for every (s, d) row of ``block_pairs``, K and V, all layers.

    One side is normally the device pool and the other a pinned host pool of the
    same per-block shape (swap-out: src on the device; swap-in: dst on the
    device). CPU tensors must be pinned; ``block_pairs`` (int64 ``[N, 2]``) may be
    on the device or pinned. Runs on ``stream`` (default: the current stream of
    the CUDA side) and returns without waiting.
    """
    cuda = [t for t in (dst_k, dst_v, src_k, src_v, block_pairs, device_error)
            if t is not None and t.is_cuda]
    if not cuda:
        raise ValueError("swap_blocks needs at least one CUDA pool (no CPU path)")
    dev = _require_cuda(*cuda)
    for name, t in (("dst_k", dst_k), ("dst_v", dst_v), ("src_k", src_k), ("src_v", src_v),
                    ("block_pairs", block_pairs)):
        if not t.is_cuda and not t.is_pinned():
            raise ValueError(f"{name} is pageable host memory; allocate it with pin_memory=True")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if dst_k.shape != dst_v.shape or src_k.shape != src_v.shape:
        raise ValueError("K and V pools must have the same shape on each side")
    if len({dst_k.dtype, dst_v.dtype, src_k.dtype, src_v.dtype}) != 1:
        raise ValueError("all four pools must share one dtype")
    dl, dn, dstride = _pool_geometry(dst_k)
    sl, sn, sstride = _pool_geometry(src_k)
    if dl != sl or dst_k.shape[-3:] != src_k.shape[-3:]:
        raise ValueError("source and destination pools differ in layers or block shape")
    if block_pairs.dtype != torch.int64 or block_pairs.dim() != 2 or block_pairs.shape[1] != 2:
        raise ValueError("block_pairs must be int64 [num_pairs, 2]")
    block_bytes = math.prod(dst_k.shape[-3:]) * dst_k.element_size()
    s = (stream or torch.cuda.current_stream(dev)).cuda_stream
    st = _lib.load().ps_swap_blocks(
        dst_k.data_ptr(), dst_v.data_ptr(), dn, dstride, src_k.data_ptr(), src_v.data_ptr(), sn,
        sstride, block_pairs.data_ptr(), block_pairs.shape[0], dl, block_bytes, int(max_ctas),
        _err_ptr(device_error), s,
    )
    _lib.check(st, "swap_blocks")


def build_slot_mapping(
    block_tables: torch.Tensor,
    ctx_before: torch.Tensor,
    q_lens: torch.Tensor,
    query_len: int,
    block_size: int,
    num_blocks: int,
    positions: bool = True,
    device_error: torch.Tensor | None = None,
    out: tuple[torch.Tensor, torch.Tensor | None] | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Slots (and positions) of a left-padded ``[B, query_len]`` step, on the device.

    Sequence b's ``q_lens[b]`` new tokens are its last rows and continue from
    ``ctx_before[b]`` cached tokens; padding rows get -1. ``out`` = existing
    int64 ``(slots, positions or None)`` buffers of ``B*query_len`` to fill.
    """
    dev = _require_cuda(block_tables, ctx_before, q_lens, device_error)
    b = ctx_before.shape[0]
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != b:
        raise ValueError("block_tables must be int32 [num_seqs, max_blocks]")
    if block_tables.stride(1) != 1:
        raise ValueError("block_tables rows must be contiguous")
    for name, t in (("ctx_before", ctx_before), ("q_lens", q_lens)):
        if t.dtype != torch.int32 or t.shape != (b,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [num_seqs]")
    if out is not None:
        slots, pos = out
        for t in (slots, pos):
            if t is not None and (t.dtype != torch.int64 or t.numel() != b * query_len or
                                  not t.is_contiguous() or t.device != dev):
                raise ValueError("out buffers must be contiguous int64 [B*query_len] on the device")
    else:
        slots = torch.empty(b * query_len, dtype=torch.int64, device=dev)
        pos = torch.empty_like(slots) if positions else None
    st = _lib.load().ps_build_slot_mapping(
        slots.data_ptr(), _ptr(pos), block_tables.data_ptr(),
        block_tables.stride(0) if b > 1 else block_tables.shape[1], ctx_before.data_ptr(),
        q_lens.data_ptr(), b, int(query_len), int(block_size), block_tables.shape[1],
        int(num_blocks), _err_ptr(device_error), _stream(dev),
    )
    _lib.check(st, "build_slot_mapping")
    return slots, pos


def decode_workspace_bytes(
    num_seqs: int, num_q_heads: int, head_dim: int, block_size: int, max_blocks_per_seq: int,
    split_tokens: int,
) -> int:
    """Bytes of split-K workspace ``paged_decode`` needs (0 if nothing is split)."""
    return int(_lib.load().ps_paged_decode_workspace_bytes(
        num_seqs, num_q_heads, head_dim, block_size, max_blocks_per_seq, split_tokens))


def selftest_wait_timeout(device_error: torch.Tensor) -> None:
    """Run the shared bounded-wait failure path once: a wait on an mbarrier that
    nothing arrives at gives up after the kernels' poll bound and ORs
    ``PS_DEVERR_TIMEOUT`` into ``device_error`` (no fault, no hang)."""
    dev = _require_cuda(device_error)
    st = _lib.load().ps_selftest_wait_timeout(_err_ptr(device_error), _stream(dev))
    _lib.check(st, "selftest_wait_timeout")


def decode_order(ctx_lens: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Longest-first launch order of a decode step (int32 [B], a permutation of
    ``range(B)``), for ``paged_decode(..., seq_order=...)``; one per step serves
    every layer."""
    dev = _require_cuda(ctx_lens, out)
    if ctx_lens.dtype != torch.int32 or ctx_lens.dim() != 1 or not ctx_lens.is_contiguous():
        raise ValueError("ctx_lens must be contiguous int32 [num_seqs]")
    b = ctx_lens.shape[0]
    if out is None:
        out = torch.empty(b, dtype=torch.int32, device=dev)
    if out.dtype != torch.int32 or out.shape != (b,) or not out.is_contiguous():
        raise ValueError("out must be contiguous int32 [num_seqs]")
    st = _lib.load().ps_paged_decode_order(ctx_lens.data_ptr(), b, out.data_ptr(), _stream(dev))
    _lib.check(st, "decode_order")
    return out


class _DecodeArgs:
    """Validated arguments shared by :func:`paged_decode` and :func:`paged_decode_append`."""

    def __init__(self, query, k_pool, v_pool, block_tables, ctx_lens, out, workspace,
                 device_error, seq_order, *extra, quantised=False):
        self.dev = _require_cuda(query, k_pool, v_pool, block_tables, ctx_lens, out, workspace,
                                 device_error, seq_order, *extra)
        if not quantised:  # the caller checks an 8-bit cache's pools with their scales
            _check_pool(k_pool, "k_pool")
            _check_pool(v_pool, "v_pool")
        shape, dtype = k_pool.shape, query.dtype
        self.nb, self.hkv, self.bs, d = shape
        self.d = d
        if not quantised and (v_pool.shape != shape or dtype != k_pool.dtype):
            raise ValueError("k_pool/v_pool/query must share shape and dtype")
        if query.dim() != 3:
            raise ValueError("query must be [num_seqs, num_q_heads, head_dim]")
        b, hq, _ = query.shape
        self.b, self.hq = b, hq
        self.qs = _check_rows(query, "query", hq, d)
        if out is None:
            self.out = query.new_empty((b, hq, d))
            self.os = hq * d
        else:
            if out.shape != (b, hq, d) or out.dtype != dtype:
                raise ValueError("out must be [num_seqs, num_q_heads, head_dim] of the query dtype")
            self.out = out
            self.os = _check_rows(out, "out", hq, d)
        table_shape = block_tables.shape
        if block_tables.dtype != torch.int32 or len(table_shape) != 2 or table_shape[0] != b:
            raise ValueError("block_tables must be int32 [num_seqs, max_blocks]")
        row, unit = block_tables.stride()
        if unit != 1:
            raise ValueError("block_tables rows must be contiguous")
        if ctx_lens.dtype != torch.int32 or ctx_lens.shape != (b,) or not ctx_lens.is_contiguous():
            raise ValueError("ctx_lens must be contiguous int32 [num_seqs]")
        self.order_ptr = None
        if seq_order is not None:
            if seq_order.dtype != torch.int32 or seq_order.shape != (b,) or \
                    not seq_order.is_contiguous():
                raise ValueError("seq_order must be contiguous int32 [num_seqs]")
            self.order_ptr = seq_order.data_ptr()
        self.max_blocks = table_shape[1]
        self.bt_stride = row if b > 1 else self.max_blocks
        self.ws_ptr, self.ws_bytes = None, 0
        if workspace is not None:
            self.ws_ptr = workspace.data_ptr()
            self.ws_bytes = workspace.nbytes


def paged_decode(
    query: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    ctx_lens: torch.Tensor,
    scale: float,
    split_tokens: int = 0,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    device_error: torch.Tensor | None = None,
    seq_order: torch.Tensor | None = None,
) -> torch.Tensor:
    """Decode attention: ``query`` [B, Hq, D] over keys ``[0, ctx_lens[b])`` of each sequence.

    ``block_tables`` is int32 [B, max_blocks] and ``ctx_lens`` int32 [B]. Returns
    ``out`` [B, Hq, D]. With ``split_tokens`` > 0, sequences longer than one
    partition are split (flash-decoding) and ``workspace`` (uint8, at least
    :func:`decode_workspace_bytes`, 256-byte aligned) receives the partials.
    ``seq_order`` (int32 [B], from :func:`decode_order`) starts the longest
    sequences first; the result does not depend on it.
    """
    a = _DecodeArgs(query, k_pool, v_pool, block_tables, ctx_lens, out, workspace, device_error,
                    seq_order)
    st = _lib.load().ps_paged_decode_ordered(
        a.out.data_ptr(), a.os, query.data_ptr(), a.qs, k_pool.data_ptr(), v_pool.data_ptr(),
        a.nb, block_tables.data_ptr(), a.bt_stride, ctx_lens.data_ptr(), a.b, a.hq, a.hkv, a.d,
        a.bs, a.max_blocks, float(scale), int(split_tokens), a.ws_ptr, a.ws_bytes,
        _dtype_code(query), a.order_ptr, _err_ptr(device_error), _stream(a.dev),
    )
    _lib.check(st, "paged_decode")
    return a.out


def paged_decode_listed(
    query: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    ctx_lens: torch.Tensor,
    seq_list: torch.Tensor,
    scale: float,
    split_tokens: int = 0,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    device_error: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`paged_decode` for the sequences in ``seq_list`` (int32 [n], indices
    into the batch, taken in that order) only; other rows of ``out`` are left
    as they are. ``query``/``out`` are [B, Hq, D] views whose rows may be strided
    (e.g. each sequence's last row of a [B, query_len, Hq, D] step)."""
    a = _DecodeArgs(query, k_pool, v_pool, block_tables, ctx_lens, out, workspace, device_error,
                    None, seq_list)
    if seq_list.dtype != torch.int32 or seq_list.dim() != 1 or not seq_list.is_contiguous():
        raise ValueError("seq_list must be contiguous int32 [n]")
    n = seq_list.shape[0]
    st = _lib.load().ps_paged_decode_listed(
        a.out.data_ptr(), a.os, query.data_ptr(), a.qs, k_pool.data_ptr(), v_pool.data_ptr(),
        a.nb, block_tables.data_ptr(), a.bt_stride, ctx_lens.data_ptr(), a.b,
        seq_list.data_ptr() if n else None, n, a.hq, a.hkv, a.d, a.bs, a.max_blocks, float(scale),
        int(split_tokens), a.ws_ptr, a.ws_bytes, _dtype_code(query), _err_ptr(device_error),
        _stream(a.dev),
    )
    _lib.check(st, "paged_decode_listed")
    return a.out


def paged_decode_quant(
    query: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    ctx_lens: torch.Tensor,
    scale: float,
    split_tokens: int = 0,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    device_error: torch.Tensor | None = None,
    seq_order: torch.Tensor | None = None,
    planned: bool = False,
    seq_list: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`paged_decode` over an 8-bit cache (:func:`cache_append_quant`).

    ``query``/``out`` are bf16 or fp16, the pools ``float8_e4m3fn`` or ``int8`` codes with
    their scales. ``split_tokens``, ``workspace`` (:func:`decode_workspace_bytes`) and
    ``seq_order`` as in :func:`paged_decode`; ``planned``: the split-K unit list of
    these lengths is already in ``workspace`` (:func:`decode_plan`); ``seq_list``: only
    these sequences, as in :func:`paged_decode_listed` (not with ``seq_order`` or
    ``planned``). Keys past a sequence's length are ignored whatever their rows hold.
    """
    code = _check_quant_pools(k_pool, v_pool, k_scale, v_scale)
    a = _DecodeArgs(query, k_pool, v_pool, block_tables, ctx_lens, out, workspace, device_error,
                    seq_order, seq_list, k_scale, v_scale, quantised=True)
    listed, list_ptr = -1, a.order_ptr
    if seq_list is not None:
        if seq_order is not None or planned:
            raise ValueError("seq_list cannot be combined with seq_order or planned")
        if seq_list.dtype != torch.int32 or seq_list.dim() != 1 or not seq_list.is_contiguous():
            raise ValueError("seq_list must be contiguous int32 [n]")
        listed = seq_list.shape[0]
        list_ptr = seq_list.data_ptr() if listed else None
    st = _launch(
        a.dev, _lib.load().ps_paged_decode_quant, a.out.data_ptr(), a.os, query.data_ptr(), a.qs,
        k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), a.nb,
        block_tables.data_ptr(), a.bt_stride, ctx_lens.data_ptr(), a.b, list_ptr, listed, a.hq,
        a.hkv, a.d, a.bs, a.max_blocks, float(scale), int(split_tokens), int(planned), a.ws_ptr,
        a.ws_bytes, _dtype_code(query), code, _err_ptr(device_error), _stream(a.dev),
    )
    _lib.check(st, "paged_decode_quant")
    return a.out


def decode_shared_workspace_bytes(
    num_seqs: int, num_q_heads: int, head_dim: int, block_size: int, max_blocks_per_seq: int,
    max_shared: int, split_keys: int, split_tokens: int,
) -> int:
    """Bytes of workspace :func:`paged_decode_shared` needs (0 if nothing is shared or split)."""
    return int(_lib.load().ps_paged_decode_shared_workspace_bytes(
        num_seqs, num_q_heads, head_dim, block_size, max_blocks_per_seq, max_shared, split_keys,
        split_tokens))


def shared_split_keys(group_sizes: list[int], num_q_heads: int, num_kv_heads: int,
                      max_shared: int, num_sms: int) -> int:
    """Keys per piece of a shared-prefix pass over groups of these sizes; 0 = one piece.

    The pass runs one unit (an item's piece) per SM at a time: an item is two 128-row query
    tiles of a group and KV head, a row being one sequence and query head, and takes a
    key tile of 128 keys a step; where every group fits one tile, its two tiles take two key
    tiles a step. A unit costs about five steps more than its keys (lookups, first loads,
    writing partials), and a partial a quarter of a step in the merge, so this picks the
    pieces (at most 64) that cost the fewest steps:
    ``waves * (steps + 5) + partials / 4``. Measured best against this choice: 256 rows over
    8192 keys 4 / 4 pieces, 8 rows of 64 heads over 32768 keys 12-16 / 16, groups of 32, 30
    and 20 over 4096, 2048 and 6000 keys 6 / 6.
    """
    if not group_sizes or max_shared <= 0 or num_sms <= 0:
        return 0
    rows = 128 // (num_q_heads // num_kv_heads)
    paired = max(group_sizes) <= rows
    items = sum(1 if paired else -(-n // (2 * rows)) for n in group_sizes) * num_kv_heads
    tiles = -(-max_shared // 128)
    best, best_cost = 0, math.inf
    for pieces in range(1, min(64, tiles) + 1):
        per_piece = -(-tiles // pieces)
        if pieces > 1 and per_piece == -(-tiles // (pieces - 1)):
            continue  # the same cut as with one piece less
        steps = -(-per_piece // 2) if paired else per_piece
        waves = -(-items * -(-tiles // per_piece) // num_sms)
        cost = waves * (steps + 5) + -(-tiles // per_piece) * (2 if paired else 1) / 4
        if cost < best_cost:
            best, best_cost = per_piece * 128, cost
    return 0 if best >= tiles * 128 else best


def paged_decode_shared(
    query: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    ctx_lens: torch.Tensor,
    group_starts: torch.Tensor,
    shared_lens: torch.Tensor,
    max_group: int,
    max_shared: int,
    scale: float,
    split_keys: int = 0,
    split_tokens: int = 0,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    device_error: torch.Tensor | None = None,
    seq_order: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`paged_decode` where neighbouring sequences share their leading blocks.

    Group g is rows ``[group_starts[g], group_starts[g + 1])`` of the batch (int32
    ``[groups + 1]``, at most ``max_group`` rows each); ``shared_lens`` (int32 [B]) gives
    each row's shared keys: whole blocks, the same for all rows of a group, at most
    ``max_shared``, 0 for rows that share nothing. A group's prefix is read once for all
    its rows, in pieces of ``split_keys`` keys (:func:`shared_split_keys`; 0 = one
    piece); the keys behind it go as in :func:`paged_decode`, cut by ``split_tokens``
    and taken in ``seq_order`` (:func:`decode_order` of ``ctx_lens - shared_lens``).
    ``workspace``: uint8, :func:`decode_shared_workspace_bytes`, allocated here when not
    given. Keys past a sequence's length are ignored whatever their rows hold.
    """
    a = _DecodeArgs(query, k_pool, v_pool, block_tables, ctx_lens, out, workspace, device_error,
                    seq_order, group_starts, shared_lens)
    if shared_lens.dtype != torch.int32 or shared_lens.shape != (a.b,) or \
            not shared_lens.is_contiguous():
        raise ValueError("shared_lens must be contiguous int32 [num_seqs]")
    if group_starts.dtype != torch.int32 or group_starts.dim() != 1 or \
            group_starts.shape[0] < 1 or not group_starts.is_contiguous():
        raise ValueError("group_starts must be contiguous int32 [num_groups + 1]")
    if workspace is None:
        need = decode_shared_workspace_bytes(a.b, a.hq, a.d, a.bs, a.max_blocks, int(max_shared),
                                             int(split_keys), int(split_tokens))
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=a.dev)
        a.ws_ptr, a.ws_bytes = workspace.data_ptr(), workspace.numel()
    st = _launch(
        a.dev, _lib.load().ps_paged_decode_shared, a.out.data_ptr(), a.os, query.data_ptr(), a.qs,
        k_pool.data_ptr(), v_pool.data_ptr(), a.nb, block_tables.data_ptr(), a.bt_stride,
        ctx_lens.data_ptr(), a.b, group_starts.data_ptr(), group_starts.shape[0] - 1,
        shared_lens.data_ptr(), int(max_group), int(max_shared), a.hq, a.hkv, a.d, a.bs,
        a.max_blocks, float(scale), int(split_keys), int(split_tokens), a.ws_ptr, a.ws_bytes,
        _dtype_code(query), a.order_ptr, _err_ptr(device_error), _stream(a.dev),
    )
    _lib.check(st, "paged_decode_shared")
    return a.out


def decode_plan(
    ctx_lens: torch.Tensor,
    workspace: torch.Tensor,
    num_q_heads: int,
    head_dim: int,
    block_size: int,
    max_blocks: int,
    split_tokens: int,
    seq_order: torch.Tensor | None = None,
) -> None:
    """Plan a split-K decode step once for all its layers (``ps_paged_decode_plan``):
    the (sequence, partition) units of ``ctx_lens`` in ``seq_order`` go into
    ``workspace``; each layer then calls :func:`paged_decode_append` with
    ``planned=True``. A no-op when ``split_tokens`` splits nothing."""
    dev = _require_cuda(ctx_lens, workspace, seq_order)
    if ctx_lens.dtype != torch.int32 or ctx_lens.dim() != 1 or not ctx_lens.is_contiguous():
        raise ValueError("ctx_lens must be contiguous int32 [num_seqs]")
    b = ctx_lens.shape[0]
    if seq_order is not None and (seq_order.dtype != torch.int32 or seq_order.shape != (b,)
                                  or not seq_order.is_contiguous()):
        raise ValueError("seq_order must be contiguous int32 [num_seqs]")
    st = _lib.load().ps_paged_decode_plan(
        ctx_lens.data_ptr(), b, seq_order.data_ptr() if seq_order is not None else None,
        num_q_heads, head_dim, block_size, max_blocks, int(split_tokens), workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), _stream(dev),
    )
    _lib.check(st, "decode_plan")


def paged_decode_append(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    ctx_lens: torch.Tensor,
    scale: float,
    split_tokens: int = 0,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    device_error: torch.Tensor | None = None,
    seq_order: torch.Tensor | None = None,
    planned: bool = False,
) -> torch.Tensor:
    """One decode step in one launch: ``cache_append`` of the step's new token
    (``key``/``value`` [B, Hkv, D], ``slot_mapping`` int64 [B], -1 = none) followed by
    :func:`paged_decode`, with the same pool contents and output. Each slot must be
    the position ``ctx_lens[b] - 1``. ``planned``: the split-K unit list for this
    step is already in ``workspace`` (:func:`decode_plan`); no plan kernel runs."""
    a = _DecodeArgs(query, k_pool, v_pool, block_tables, ctx_lens, out, workspace, device_error,
                    seq_order, key, value, slot_mapping)
    for t, name in ((key, "key"), (value, "value")):
        if t.dtype != k_pool.dtype or t.dim() != 3 or t.shape[0] != a.b:
            raise ValueError(f"{name} must be [num_seqs, num_kv_heads, head_dim] of the pool dtype")
    ks = _check_rows(key, "key", a.hkv, a.d)
    vs = _check_rows(value, "value", a.hkv, a.d)
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (a.b,) or \
            not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int64 [num_seqs]")
    lib = _lib.load()
    fn = lib.ps_paged_decode_append_planned if planned else lib.ps_paged_decode_append
    st = fn(
        a.out.data_ptr(), a.os, query.data_ptr(), a.qs, key.data_ptr(), ks, value.data_ptr(), vs,
        slot_mapping.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), a.nb,
        block_tables.data_ptr(), a.bt_stride, ctx_lens.data_ptr(), a.b, a.hq, a.hkv, a.d, a.bs,
        a.max_blocks, float(scale), int(split_tokens), a.ws_ptr, a.ws_bytes, _dtype_code(query),
        a.order_ptr, _err_ptr(device_error), _stream(a.dev),
    )
    _lib.check(st, "paged_decode_append")
    return a.out


def prefill_workspace_bytes(
    num_seqs: int, max_q_len: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
    block_size: int, max_blocks_per_seq: int, split_keys: int,
) -> int:
    """Bytes of workspace ``paged_prefill(..., split_keys=...)`` needs (0 if nothing is split)."""
    return int(_lib.load().ps_paged_prefill_workspace_bytes(
        num_seqs, max_q_len, num_q_heads, num_kv_heads, head_dim, block_size,
        max_blocks_per_seq, split_keys))


def prefill_split_keys(num_items: int, max_keys: int, num_sms: int, min_piece_keys: int = 512,
                       max_pieces: int = 16) -> int:
    """Keys per split-K piece for a prefill of ``num_items`` work items (query-tile
    pairs x KV heads, each two tiles of 128 query rows) over at most ``max_keys``
    keys each; 0 runs every item whole.

    The prefill kernel runs one persistent CTA per SM, so fewer items than two
    waves of ``num_sms`` leave SMs idle, or a last wave half full, while each item
    walks its whole context. Cutting every item into ``pieces`` key ranges of at
    least ``min_piece_keys`` keys makes ``num_items * pieces`` units: this picks
    the fewest pieces whose units fill whole waves to 90% or more (else the best
    fill found), and no split when one piece is best.
    """
    if num_items <= 0 or num_items >= 2 * num_sms or num_sms <= 0:
        return 0
    tiles = -(-max_keys // 128)
    limit = min(max_pieces, tiles * 128 // max(min_piece_keys, 128))
    best, best_fill = 1, 0.0
    for pieces in range(1, limit + 1):
        units = num_items * pieces
        fill = units / (-(-units // num_sms) * num_sms)
        if fill > best_fill + 1e-9:
            best, best_fill = pieces, fill
        if fill >= 0.9:
            best = pieces
            break
    if best == 1:
        return 0
    return -(-tiles // best) * 128


def paged_prefill(
    query: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    q_starts: torch.Tensor,
    q_lens: torch.Tensor,
    ctx_lens: torch.Tensor,
    max_q_len: int,
    scale: float,
    out: torch.Tensor | None = None,
    device_error: torch.Tensor | None = None,
    split_keys: int = 0,
    workspace: torch.Tensor | None = None,
    max_keys: int | None = None,
) -> torch.Tensor:
    """Causal paged prefill over cached prefix + new tokens.

    ``query``/``out`` are [rows, Hq, D]; sequence b owns rows
    ``[q_starts[b], q_starts[b] + q_lens[b])`` and its query i attends keys
    ``[0, ctx_lens[b] + i]`` read through ``block_tables``. The new tokens' K/V
    must already be in the pools. Rows owned by no sequence are left untouched.

    ``split_keys`` > 0 cuts each work item's key range into pieces of that many
    keys (a multiple of 128) run by different CTAs and merged by a second launch
    (ps_paged_prefill_split), for prefills with few query tiles over long
    contexts. ``max_keys`` (context + new tokens of the longest sequence) bounds
    the pieces per item and so the workspace; by default the table width does.
    ``workspace`` (uint8, ``prefill_workspace_bytes`` of the same sizes) is
    allocated here when not given.
    """
    dev = _require_cuda(query, k_pool, v_pool, block_tables, q_starts, q_lens, ctx_lens, out,
                        device_error)
    _check_pool(k_pool, "k_pool")
    _check_pool(v_pool, "v_pool")
    nb, hkv, bs, d = k_pool.shape
    if v_pool.shape != k_pool.shape or query.dtype != k_pool.dtype:
        raise ValueError("k_pool/v_pool/query must share shape and dtype")
    if query.dim() != 3:
        raise ValueError("query must be [rows, num_q_heads, head_dim]")
    rows, hq, _ = query.shape
    qs = _check_rows(query, "query", hq, d)
    if out is None:
        out = torch.zeros((rows, hq, d), dtype=query.dtype, device=dev)
    if out.shape != (rows, hq, d) or out.dtype != query.dtype:
        raise ValueError("out must match query")
    os_ = _check_rows(out, "out", hq, d)
    b = q_starts.shape[0]
    for name, t in (("q_starts", q_starts), ("q_lens", q_lens), ("ctx_lens", ctx_lens)):
        if t.dtype != torch.int32 or t.shape != (b,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [num_seqs]")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != b:
        raise ValueError("block_tables must be int32 [num_seqs, max_blocks]")
    if block_tables.stride(1) != 1:
        raise ValueError("block_tables rows must be contiguous")
    width = block_tables.shape[1]
    max_blocks = width
    if max_keys is not None:
        max_blocks = max(1, min(width, -(-int(max_keys) // bs)))
    bt_stride = block_tables.stride(0) if b > 1 else width
    lib = _lib.load()
    if split_keys:
        need = prefill_workspace_bytes(b, int(max_q_len), hq, hkv, d, bs, max_blocks,
                                       int(split_keys))
        if workspace is None:
            workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
        _require_cuda(workspace)
        if workspace.device != dev or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous buffer on the query's device")
        st = lib.ps_paged_prefill_split(
            out.data_ptr(), os_, query.data_ptr(), qs, rows, k_pool.data_ptr(),
            v_pool.data_ptr(), nb, block_tables.data_ptr(), bt_stride, q_starts.data_ptr(),
            q_lens.data_ptr(), ctx_lens.data_ptr(), b, int(max_q_len), hq, hkv, d, bs, max_blocks,
            float(scale), int(split_keys), workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), _dtype_code(query),
            _err_ptr(device_error), _stream(dev),
        )
        _lib.check(st, "paged_prefill_split")
        return out
    st = lib.ps_paged_prefill(
        out.data_ptr(), os_, query.data_ptr(), qs, rows, k_pool.data_ptr(), v_pool.data_ptr(), nb,
        block_tables.data_ptr(), bt_stride, q_starts.data_ptr(), q_lens.data_ptr(),
        ctx_lens.data_ptr(), b, int(max_q_len), hq, hkv, d, bs, max_blocks, float(scale),
        _dtype_code(query), _err_ptr(device_error), _stream(dev),
    )
    _lib.check(st, "paged_prefill")
    return out


def stream_read(buf: torch.Tensor, checksum: torch.Tensor, method: int = _lib.PS_STREAM_BULK,
                device_error: torch.Tensor | None = None) -> None:
    """Read ``buf`` once (diagnostic HBM read stream) and XOR its 32-bit words into
    ``checksum`` (int32 [1] on the same device, zeroed by the caller).

    ``method``: ``PS_STREAM_BULK`` (bulk asynchronous copies into shared memory)
    or ``PS_STREAM_LOADS`` (16-byte loads from every thread).
    """
    dev = _require_cuda(buf, checksum, device_error)
    if not buf.is_contiguous() or checksum.dtype != torch.int32 or checksum.numel() < 1:
        raise ValueError("buf must be contiguous; checksum int32 [1]")
    nbytes = buf.numel() * buf.element_size()
    lib = _lib.load()
    st = lib.ps_stream_read(buf.data_ptr(), nbytes, checksum.data_ptr(), method,
                            _err_ptr(device_error), _stream(dev))
    _lib.check(st, "stream_read")
