"""Dense 8-bit block KV cache: its tables, store, read-back and attention.

The cache that keeps every token, beside the compact one that DMS evicts from
(the reference's dense paged path, attention.py:17-37, 94-100, keeps bf16 rows
and calls a library for attention).  Blocks of ``block_size`` tokens (a power of two,
16 .. 256) hold each kv head's rows in 8 bits with one scale per (block, head)
for K and one for V:

    k_cache [blocks, heads, block_size, D]          int8 or float8_e4m3fn
    v_cache [blocks, heads, block_size / 16, D, 16] V in transposed 16-token tiles
    k_scale, v_scale [blocks, heads]                fp32

A code stands for code * scale; the store's scales are powers of two.  A step
runs ``prepare_block_tables`` once, then per layer ``store_block_kvcache`` and
``block_attention``; ``gather_block_kvcache`` reads rows back dense, e.g. to
pack a prompt into the compact layout.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .. import _native as nat

TILE = 16            # tokens per transposed V tile
MAX_SEQS = 4096      # sequences per prepare_block_tables call
BLOCK_SIZES = (16, 32, 64, 128, 256)
CACHE_DTYPES = (torch.int8, torch.float8_e4m3fn)
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_INT_MAX = 2 ** 31 - 1

# bits of BlockTables.status
STATUS_NO_BLOCKS, STATUS_TABLE_WIDTH, STATUS_NUM_TOKENS, STATUS_INVALID = 1, 2, 4, 8


class BlockTables(NamedTuple):
    """A step's metadata, on the device (prepare_block_tables)."""
    slot_mapping: torch.Tensor   # int32 [num_tokens], -1 past the step's last token
    positions: torch.Tensor      # int64 [num_tokens], 0 past the step's last token
    cu_seqlens: torch.Tensor     # int32 [seqs + 1]
    context_lens: torch.Tensor   # int32 [seqs], cached + new
    free_count: torch.Tensor     # int32 [1], what is left of the stack
    status: torch.Tensor         # int32 [1], 0 or STATUS_* bits


def allocate_block_kvcache(num_blocks: int, num_kv_heads: int, block_size: int, head_dim: int,
                           dtype: torch.dtype = torch.int8, device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale) of ``num_blocks`` blocks; the codes
    are not initialised."""
    if dtype not in CACHE_DTYPES:
        raise ValueError(f"a block KV cache holds int8 or float8_e4m3fn, got {dtype}")
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
    if head_dim not in (64, 128):
        raise ValueError(f"the block KV cache supports head_dim 64 or 128, got {head_dim}")
    if num_blocks < 1 or num_kv_heads < 1 or num_blocks * block_size > _INT_MAX:
        raise ValueError("a block KV cache needs at least one block and head and fewer than 2^31 slots")
    k = torch.empty((num_blocks, num_kv_heads, block_size, head_dim), device=device, dtype=dtype)
    v = torch.empty((num_blocks, num_kv_heads, block_size // TILE, head_dim, TILE), device=device, dtype=dtype)
    return (k, v, torch.zeros((num_blocks, num_kv_heads), device=device),
            torch.zeros((num_blocks, num_kv_heads), device=device))


def _check_cache(k_cache, v_cache, k_scale, v_scale) -> tuple[int, int, int, int]:
    """(blocks, heads, block size, head_dim) of a well-formed cache."""
    if k_cache.dtype not in CACHE_DTYPES or v_cache.dtype != k_cache.dtype:
        raise ValueError(f"a block KV cache holds int8 or float8_e4m3fn, got {k_cache.dtype} / {v_cache.dtype}")
    if k_cache.ndim != 4:
        raise ValueError(f"expected k_cache [blocks, heads, block_size, head_dim], got {tuple(k_cache.shape)}")
    nb, h, bs, d = k_cache.shape
    if bs not in BLOCK_SIZES or d not in (64, 128):
        raise ValueError(f"block_size must be one of {BLOCK_SIZES} and head_dim 64 or 128, got {bs} and {d}")
    if v_cache.shape != (nb, h, bs // TILE, d, TILE):
        raise ValueError(f"expected v_cache {(nb, h, bs // TILE, d, TILE)}, got {tuple(v_cache.shape)}")
    if nb < 1 or nb * bs > _INT_MAX:
        raise ValueError("a block KV cache needs at least one block and fewer than 2^31 slots")
    kb, kh, kr, kd = k_cache.stride()
    vb, vh, vt, vd, vi = v_cache.stride()
    if kd != 1 or kr != d or vi != 1 or vd != TILE or (bs > TILE and vt != TILE * d):
        raise ValueError("a head's part of a block must be contiguous in k_cache and v_cache")
    if (kb | kh | vb | vh | k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise ValueError("k_cache and v_cache blocks must be 16-byte aligned")
    if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32 or \
            k_scale.shape != (nb, h) or v_scale.shape != (nb, h):
        raise ValueError(f"expected fp32 scales [{nb}, {h}], got {k_scale.dtype} {tuple(k_scale.shape)} and "
                         f"{v_scale.dtype} {tuple(v_scale.shape)}")
    sb, sh = k_scale.stride()
    tb, th = v_scale.stride()
    if h > 1 and (sh != 1 or th != 1) or nb > 1 and sb != tb:
        raise ValueError("k_scale and v_scale need contiguous heads and the same block stride")
    return nb, h, bs, d


def _device_index(what: str, *tensors) -> int:
    """The index of the one GPU that holds all tensors."""
    i = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != i or i < 0:
            raise RuntimeError(f"{what} requires its tensors on one GPU (HIP device); got {t.device} and "
                               f"{tensors[0].device}")
    return i


def _launch(index: int, name: str, *args) -> None:
    """nat.call on the tensors' device, on its current stream."""
    if index == torch.cuda.current_device():
        nat.call(name, *args, nat.raw_stream(index))
    else:
        with torch.cuda.device(index):
            nat.call(name, *args, nat.raw_stream(index))


def _int32(what: str, t: torch.Tensor, shape: tuple) -> None:
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 {list(shape)} tensor, got {t.dtype} {list(t.shape)}")


def _overlap(outs, ins) -> bool:
    """Whether the memory of one of the contiguous ``outs`` meets an input's span."""
    spans = []
    for x in ins:
        if x.numel():
            size = 1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
            spans.append((x.data_ptr(), x.data_ptr() + size * x.element_size()))
    for o in outs:
        start, end = o.data_ptr(), o.data_ptr() + o.numel() * o.element_size()
        if any(start < b and a < end for a, b in spans):
            return True
    return False


def prepare_block_tables(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor,
                         free_blocks: torch.Tensor, free_count: torch.Tensor, *, block_size: int, num_tokens: int,
                         out: BlockTables | None = None) -> BlockTables:
    """Block tables and slot map of a step, on the device from its lengths.

    Sequence b holds ``cached_lens[b]`` tokens in the first
    ``ceil(cached / block_size)`` entries of ``block_tables[b]`` and gets
    ``new_lens[b]`` (0 or more) in this step.  The blocks it lacks are popped
    from the stack ``free_blocks[: free_count]``, top first, in the order of
    the sequences, and written into its table row.  Token t of the step,
    sequence after sequence, gets its position and its slot
    ``table[position // block_size] * block_size + position % block_size``;
    ``num_tokens`` is the length of those outputs and may exceed the step's
    tokens (a padded batch).  Nothing is read back: the host passes sizes only.

    When the stack, a table row or ``num_tokens`` is too short, or a length or
    the count is invalid, ``status`` says so (STATUS_* bits) and nothing is
    popped: the tables stay, every slot is -1, cu_seqlens is 0 and context_lens
    the cached lengths.  ``free_count`` is not changed in place, so a step can
    be prepared again; ``out`` takes an earlier call's tensors (captured steps),
    which share no memory with the arguments: the launch's workgroups read those
    while others write."""
    n = cached_lens.numel()
    if not 1 <= n <= MAX_SEQS:
        raise ValueError(f"prepare_block_tables takes 1 to {MAX_SEQS} sequences, got {n}")
    _int32("cached_lens", cached_lens, (n,))
    _int32("new_lens", new_lens, (n,))
    _int32("free_blocks", free_blocks, (free_blocks.numel(),))
    _int32("free_count", free_count, (1,))
    if block_tables.dtype != torch.int32 or block_tables.ndim != 2 or block_tables.shape[0] != n:
        raise ValueError(f"block_tables must be int32 [{n}, blocks], got {block_tables.dtype} "
                         f"{tuple(block_tables.shape)}")
    width = block_tables.shape[1]
    if width > 1 and block_tables.stride(1) != 1 or n > 1 and block_tables.stride(0) < width:
        raise ValueError("block_tables needs rows of its own with contiguous entries")
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
    if not 0 <= num_tokens <= _INT_MAX:
        raise ValueError(f"num_tokens must be between 0 and {_INT_MAX}, got {num_tokens}")
    if out is not None:
        for what, size in (("slot_mapping", num_tokens), ("cu_seqlens", n + 1), ("context_lens", n),
                           ("free_count", 1), ("status", 1)):
            _int32(f"out.{what}", getattr(out, what), (size,))
        if out.positions.dtype != torch.int64 or out.positions.shape != (num_tokens,) or \
                not out.positions.is_contiguous():
            raise ValueError(f"out.positions must be a contiguous int64 [{num_tokens}] tensor")
        if _overlap(out, (cached_lens, new_lens, block_tables, free_blocks, free_count)):
            raise ValueError("out's tensors must not share memory with the lengths, tables, free list or count")
    dev = _device_index("prepare_block_tables", cached_lens, new_lens, block_tables, free_blocks, free_count,
                        *(() if out is None else out))
    if out is None:
        slots, cu, ctx, count, status = torch.split_with_sizes(
            cached_lens.new_empty(num_tokens + 2 * n + 3), (num_tokens, n + 1, n, 1, 1))
        out = BlockTables(slots, cached_lens.new_empty(num_tokens, dtype=torch.int64), cu, ctx, count, status)
    _launch(dev, "fdms_block_tables", cached_lens.data_ptr(), new_lens.data_ptr(), n, block_tables.data_ptr(),
            block_tables.stride(0), width, free_blocks.data_ptr(), free_blocks.numel(), free_count.data_ptr(),
            block_size, num_tokens, out.slot_mapping.data_ptr(), out.positions.data_ptr(), out.cu_seqlens.data_ptr(),
            out.context_lens.data_ptr(), out.free_count.data_ptr(), out.status.data_ptr())
    return out


def _aligned_rows(x: torch.Tensor) -> torch.Tensor:
    """x [rows, heads, D] with a contiguous head_dim and 16-byte aligned rows: itself, or a copy."""
    st, sh, sd = x.stride()
    if sd == 1 and not ((st | sh) * x.element_size() | x.data_ptr()) % 16:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _codes(k_cache, v_cache) -> tuple:
    """(k, v, is_fp8, block and head strides) as the C entry points take a cache's codes."""
    kb, kh = k_cache.stride()[:2]
    vb, vh = v_cache.stride()[:2]
    return k_cache.data_ptr(), v_cache.data_ptr(), int(k_cache.dtype is not torch.int8), kb, kh, vb, vh


def store_block_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Store rows key / value [T, heads, D] (fp32, fp16 or bf16) at their slots.

    ``slot_mapping`` int32 [T] as prepare_block_tables writes it: the rows a
    call brings to one block are neighbours with consecutive slots and follow
    the rows that the block holds already (a call whose rows reach one block in
    several runs leaves that block's contents undefined).  A slot that is
    negative or past the cache is skipped.

    Per (block, head) the scale is the least power of two s with
    ``max |x| <= 127 s`` (int8) or ``448 s`` (e4m3fn) over the new rows, at
    least 2^-126, and no less than the block's scale if it held rows before;
    codes are x / s rounded to nearest even.  When new rows raise the scale,
    the earlier rows' codes are rounded again to it.  Infinities saturate
    (counting as the largest fp32 value for the scale) and NaN is stored as 0:
    a cached row never poisons another sequence position's attention."""
    nb, h, bs, d = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if key.ndim != 3 or key.shape != value.shape or key.shape[1:] != (h, d):
        raise ValueError(f"expected key and value [tokens, {h}, {d}], got {tuple(key.shape)} and "
                         f"{tuple(value.shape)}")
    if key.dtype not in _FLOATS or value.dtype != key.dtype:
        raise ValueError(f"key and value must be fp32, fp16 or bf16 alike, got {key.dtype} and {value.dtype}")
    if k_scale.data_ptr() == v_scale.data_ptr() or nb > 1 and 0 in (k_cache.stride(0), v_cache.stride(0),
                                                                    k_scale.stride(0)) or \
            h > 1 and 0 in (k_cache.stride(1), v_cache.stride(1)):
        raise ValueError("K and V, blocks and heads need memory of their own to be stored into")
    t = key.shape[0]
    _int32("slot_mapping", slot_mapping, (t,))
    dev = _device_index("store_block_kvcache", key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
    if t == 0:
        return
    key, value = _aligned_rows(key), _aligned_rows(value)
    kst, ksh, _ = key.stride()
    vst, vsh, _ = value.stride()
    _launch(dev, "fdms_store_block_kvcache", key.data_ptr(), value.data_ptr(), nat.dtype_code(key.dtype), kst, ksh,
            vst, vsh, *_codes(k_cache, v_cache), k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0),
            slot_mapping.data_ptr(), t, nb, bs, h, d)


def gather_block_kvcache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                         slot_mapping: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """Dense (K, V) [T, heads, D] of the rows at ``slot_mapping`` int32 [T]:
    code * scale, exact in bf16 and fp32 for the store's scales.  Any slots in
    any order; one that is negative or past the cache gives a row of zeros."""
    nb, h, bs, d = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if dtype not in _FLOATS:
        raise ValueError(f"gather_block_kvcache returns fp32, fp16 or bf16, not {dtype}")
    t = slot_mapping.numel()
    _int32("slot_mapping", slot_mapping, (t,))
    dev = _device_index("gather_block_kvcache", k_cache, v_cache, k_scale, v_scale, slot_mapping)
    k = slot_mapping.new_empty((t, h, d), dtype=dtype)
    v = slot_mapping.new_empty((t, h, d), dtype=dtype)
    if t:
        _launch(dev, "fdms_gather_block_kvcache", *_codes(k_cache, v_cache), k_scale.data_ptr(), v_scale.data_ptr(),
                k_scale.stride(0), slot_mapping.data_ptr(), t, nb, bs, h, d, k.data_ptr(), v.data_ptr(),
                nat.dtype_code(dtype), h * d, d, h * d, d)
    return k, v


def block_attention_plan(seqs: int, heads: int, group: int, rows: int, max_seqlen: int,
                         max_context: int) -> tuple[int, int, int, int]:
    """(few_rows, few_splits, few_share, tile_splits) of a block_attention
    launch over ``rows`` query rows: sequences of up to few_rows rows go to the
    kernel for few rows, longer ones to the one for many; 0 splits leave a
    launch out.

    A batch whose longest run has at most 32 rows x heads takes the first
    kernel alone, one sequence of more the second alone; several sequences may
    be of both kinds, and the first then takes those of at most 16.  Splits:
    the first kernel cuts every context into pieces of few_share 64-key groups,
    as many as give three workgroups per CU if all were the longest, between 4
    and 32 (more where that would make over 256 pieces of a context, or over 8192
    in all); the second those, each of at least 512 keys, for which the least
    time is expected: keys per split times the turns that the tiles' workgroups
    take at 512 at a time (between whole turns, as equal ones need, and the
    even share that unequal ones approach), and what a part more to write and
    join costs (777 queries over 30 000 tokens, 32 / 8 heads of 128, 1 to 5
    parts: 659, 504, 547, 528, 454 us; a chunk of 1 000 among 15 decoding
    sequences: 138, 130, 128, 140, 145)."""
    pairs = seqs * heads
    if max_seqlen * group <= 32:
        few_rows = max_seqlen
    else:
        few_rows = 16 // group if seqs > 1 else 0
    groups = -(-max_context // 64)
    share = max(min(32, max(4, -(-groups * pairs // 768))), -(-groups // 256), -(-groups * pairs // 8192))
    few = max(1, -(-groups // share)) if few_rows else 0
    if few_rows >= max_seqlen:
        return few_rows, few, share, 0
    tiles = heads * -(-rows * group // 128)
    most = max(1, min(-(-max_context // 512), 16)) if tiles < 1024 else 1

    def cost(n: int) -> float:
        turns = tiles * n / 512
        return (0.5 * -(-tiles * n // 512) + 0.5 * (turns + 0.5)) / n + 1000 / max(max_context, 1) * n

    return few_rows, few, share, min(range(1, most + 1), key=cost)


def block_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, *,
                    cu_seqlens: torch.Tensor | None = None, max_seqlen: int = 1, max_context: int | None = None,
                    scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention of q [T, q heads, D] (bf16 or fp16) over the cache.

    Sequence b's keys are the ``context_lens[b]`` rows its ``block_tables``
    row leads to and its queries rows ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1``
    of q, the last of its keys (bottom-right causal alignment, as
    ``prefill_attention``); without ``cu_seqlens`` row b is sequence b's one
    query.  ``max_seqlen`` bounds a sequence's queries and ``max_context`` the
    contexts (default: what a table row can hold); both are host numbers that
    shape the launch.  A query that sees no key gets zeros, rows past
    ``cu_seqlens[-1]`` of ``out`` are left as they are, and keys of a block
    that is not in the cache are left out.  Default ``scale`` (any finite
    number): D ** -0.5.  The cache's scales must not be negative; those that
    are not powers of two are taken exactly for the queries of few-row
    sequences, and else codes times scales are rounded to 2^-10 of themselves."""
    nb, h, bs, d = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if q.ndim != 3 or q.shape[2] != d or q.shape[1] % h or q.shape[1] == 0:
        raise ValueError(f"expected q [rows, a multiple of {h} heads, {d}], got {tuple(q.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"block attention expects bf16 or fp16 q, got {q.dtype}")
    t, hq = q.shape[:2]
    n = context_lens.numel()
    _int32("context_lens", context_lens, (n,))
    if block_tables.dtype != torch.int32 or block_tables.ndim != 2 or block_tables.shape[0] != n or n == 0:
        raise ValueError(f"block_tables must be int32 [{n}, blocks] for at least one sequence, got "
                         f"{block_tables.dtype} {tuple(block_tables.shape)}")
    width = block_tables.shape[1]
    if width > 1 and block_tables.stride(1) != 1:
        raise ValueError("block_tables needs rows with contiguous entries")
    if cu_seqlens is not None:
        _int32("cu_seqlens", cu_seqlens, (n + 1,))
    elif t != n or max_seqlen != 1:
        raise ValueError(f"without cu_seqlens q has one row per sequence, got {t} rows for {n} sequences and "
                         f"max_seqlen {max_seqlen}")
    max_seqlen = int(max_seqlen)
    if max_seqlen < 1:
        raise ValueError(f"max_seqlen must be at least 1, got {max_seqlen}")
    max_context = width * bs if max_context is None else int(max_context)
    if max_context < 0:
        raise ValueError(f"max_context must not be negative, got {max_context}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    if out is None:
        out = q.new_empty((t, hq, d))
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or \
            (out.stride(0) | out.stride(1)) % 4 or out.data_ptr() % 8:
        raise ValueError("out must have q's shape and type, a contiguous head_dim and 8-byte aligned rows")
    dev = _device_index("block_attention", q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, out,
                        *(() if cu_seqlens is None else (cu_seqlens,)))
    if t == 0:
        return out
    q = _aligned_rows(q)
    few_rows, few_splits, few_share, tile_splits = block_attention_plan(n, h, hq // h, t, max_seqlen, max_context)
    # the splits' parts, the call's own: nothing is shared between streams or captured graphs
    room = few_splits * n * few_rows * hq * (d + 2) if few_splits > 1 else 0
    if tile_splits > 1:
        room += t * hq * (tile_splits * (d + 2) + 1)
    ws = k_scale.new_empty(room) if room else None
    qst, qsh, _ = q.stride()
    ost, osh, _ = out.stride()
    _launch(dev, "fdms_block_attention", q.data_ptr(), nat.dtype_code(q.dtype), qst, qsh, t,
            *_codes(k_cache, v_cache), k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0),
            block_tables.data_ptr(), block_tables.stride(0), width, context_lens.data_ptr(), nat.ptr(cu_seqlens),
            out.data_ptr(), ost, osh, nat.ptr(ws), n, h, hq // h, d, nb, bs, max_seqlen, few_rows, few_splits,
            few_share, tile_splits, scale)
    return out
