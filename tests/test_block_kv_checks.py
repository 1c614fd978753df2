"""What the block KV cache's entry points refuse, on the CPU: the wrappers'
ValueErrors before any launch, and the library's own hipErrorInvalidValue."""
import ctypes

import pytest
import torch

from fastdms_amd import _native
from fastdms_amd.layers import block_kv as kv

I32 = torch.int32


def _cache(nb=3, h=2, bs=16, d=64, dtype=torch.int8):
    return kv.allocate_block_kvcache(nb, h, bs, d, dtype, "cpu")


def _tables(**change):
    a = dict(cached_lens=torch.zeros(2, dtype=I32), new_lens=torch.ones(2, dtype=I32),
             block_tables=torch.zeros((2, 4), dtype=I32), free_blocks=torch.zeros(5, dtype=I32),
             free_count=torch.zeros(1, dtype=I32), block_size=16, num_tokens=2)
    a.update(change)
    return kv.prepare_block_tables(**a)


@pytest.mark.parametrize("change", [
    dict(cached_lens=torch.zeros(2, dtype=torch.int64)),
    dict(new_lens=torch.zeros(3, dtype=I32)),
    dict(cached_lens=torch.zeros(4, dtype=I32)[::2]),
    dict(cached_lens=torch.zeros(0, dtype=I32), new_lens=torch.zeros(0, dtype=I32),
         block_tables=torch.zeros((0, 4), dtype=I32)),
    dict(cached_lens=torch.zeros(4097, dtype=I32), new_lens=torch.zeros(4097, dtype=I32),
         block_tables=torch.zeros((4097, 1), dtype=I32)),
    dict(block_tables=torch.zeros((3, 4), dtype=I32)),
    dict(block_tables=torch.zeros((2, 4), dtype=torch.int64)),
    dict(block_tables=torch.zeros((4, 2), dtype=I32).t()),
    dict(block_tables=torch.zeros((1, 4), dtype=I32).expand(2, 4)),  # two sequences, one row
    dict(free_blocks=torch.zeros(5, dtype=torch.int64)),
    dict(free_count=torch.zeros(2, dtype=I32)),
    dict(block_size=24), dict(block_size=8), dict(block_size=512),
    dict(num_tokens=-1), dict(num_tokens=2 ** 31),
])
def test_block_tables_refuse(change):
    with pytest.raises(ValueError):
        _tables(**change)


def test_block_tables_out_must_fit():
    def out(**change):
        a = dict(slot_mapping=torch.zeros(2, dtype=I32), positions=torch.zeros(2, dtype=torch.int64),
                 cu_seqlens=torch.zeros(3, dtype=I32), context_lens=torch.zeros(2, dtype=I32),
                 free_count=torch.zeros(1, dtype=I32), status=torch.zeros(1, dtype=I32))
        a.update(change)
        return kv.BlockTables(**a)
    # (CPU tensors end at the device check, after every check of shapes)
    with pytest.raises(RuntimeError):
        _tables(out=out())


def test_block_tables_out_must_not_meet_the_inputs():
    """Outputs in the inputs' memory (an in-place step) are refused, neighbours in one buffer are not."""
    def out(**change):
        a = dict(slot_mapping=torch.zeros(2, dtype=I32), positions=torch.zeros(2, dtype=torch.int64),
                 cu_seqlens=torch.zeros(3, dtype=I32), context_lens=torch.zeros(2, dtype=I32),
                 free_count=torch.zeros(1, dtype=I32), status=torch.zeros(1, dtype=I32))
        a.update(change)
        return kv.BlockTables(**a)
    buf = torch.zeros(16, dtype=I32)
    for argument, mine, field, theirs in (
            ("cached_lens", buf[:2], "context_lens", buf[:2]), ("new_lens", buf[:2], "context_lens", buf[1:3]),
            ("cached_lens", buf[2:4], "cu_seqlens", buf[:3]), ("free_count", buf[:1], "free_count", buf[:1]),
            ("free_count", buf[:1], "status", buf[:1]), ("free_blocks", buf[:5], "slot_mapping", buf[3:5]),
            ("block_tables", buf[:14].view(2, 7)[:, :4], "context_lens", buf[9:11]),
            ("free_blocks", buf[:5], "positions", buf[2:6].view(torch.int64))):
        with pytest.raises(ValueError, match="share memory"):
            _tables(**{argument: mine}, out=out(**{field: theirs}))
    with pytest.raises(RuntimeError):  # (the device check, after every other)
        _tables(cached_lens=buf[:2], new_lens=buf[2:4], out=out(context_lens=buf[4:6], cu_seqlens=buf[6:9]))


def test_library_refuses_tables_that_meet():
    if not _native.LIB_PATH.exists():
        pytest.skip("library not built")
    p = [ctypes.c_void_p(i << 12) for i in range(1, 16)]

    def tables(cached=p[0], table=p[2], free=p[3], count=p[4], slots=p[5], cu=p[7], ctx=p[8], status=p[10]):
        return _native.lib().fdms_block_tables(cached, p[1], 2, table, 5, 4, free, 1, count, 16, 1024, slots, p[6], cu,
                                               ctx, p[9], status, None)
    for bad in (dict(ctx=p[0]), dict(ctx=p[1]), dict(cu=p[4]), dict(status=p[4]), dict(status=p[3]),
                dict(ctx=ctypes.c_void_p(p[2].value + 32)), dict(cached=ctypes.c_void_p(p[5].value + 4092))):
        assert tables(**bad) == 1, bad


@pytest.mark.parametrize("op", ["tables", "store", "gather", "attention"])
def test_cpu_tensors_are_refused(op):
    c = _cache()
    with pytest.raises(RuntimeError, match="one GPU"):
        if op == "tables":
            _tables()
        elif op == "store":
            kv.store_block_kvcache(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), *c, torch.zeros(3, dtype=I32))
        elif op == "gather":
            kv.gather_block_kvcache(*c, torch.zeros(3, dtype=I32))
        else:
            _attend()


@pytest.mark.parametrize("args", [(0, 1, 16, 64), (1, 0, 16, 64), (1, 1, 48, 64), (1, 1, 16, 96), (2 ** 27, 1, 16, 64)])
def test_allocate_refuses(args):
    with pytest.raises(ValueError):
        kv.allocate_block_kvcache(*args, device="meta")
    with pytest.raises(ValueError):
        kv.allocate_block_kvcache(1, 1, 16, 64, torch.bfloat16, "meta")


def _bad_caches():
    k, v, ks, vs = _cache()
    f8 = torch.float8_e4m3fn
    yield k.bfloat16(), v, ks, vs
    yield k.view(f8), v, ks, vs
    yield k[0], v, ks, vs
    yield k[..., :48], v, ks, vs
    yield k, v.transpose(3, 4), ks, vs
    yield k, v[:2], ks, vs
    yield k, v, ks.double(), vs
    yield k, v, ks[:2], vs
    yield k, v, ks.t().contiguous().t(), vs
    yield k, v, torch.zeros((3, 4))[:, :2], vs  # another block stride than v_scale's
    yield k[:0], v[:0], ks[:0], vs[:0]
    wide = torch.zeros((3, 2, 16, 80), dtype=torch.int8)
    yield wide[..., :64], v, ks, vs            # rows that are not contiguous
    odd = torch.zeros(3 * 2 * 16 * 64 + 16, dtype=torch.int8)[8:8 + 3 * 2 * 16 * 64].view(3, 2, 16, 64)
    if odd.data_ptr() % 16:
        yield odd, v, ks, vs
    yield torch.zeros((3, 2, 24, 64), dtype=torch.int8), v, ks, vs


@pytest.mark.parametrize("i", range(len(list(_bad_caches()))))
def test_malformed_caches_are_refused(i):
    c = list(_bad_caches())[i]
    slots = torch.zeros(3, dtype=I32)
    with pytest.raises(ValueError):
        kv.gather_block_kvcache(*c, slots)
    with pytest.raises(ValueError):
        kv.store_block_kvcache(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), *c, slots)
    with pytest.raises(ValueError):
        kv.block_attention(torch.zeros(1, 4, 64, dtype=torch.bfloat16), *c, torch.zeros((1, 2), dtype=I32),
                           torch.zeros(1, dtype=I32))


@pytest.mark.parametrize("key,value,slots", [
    (torch.zeros(3, 2, 64), torch.zeros(2, 2, 64), torch.zeros(3, dtype=I32)),
    (torch.zeros(3, 1, 64), torch.zeros(3, 1, 64), torch.zeros(3, dtype=I32)),
    (torch.zeros(3, 128), torch.zeros(3, 128), torch.zeros(3, dtype=I32)),
    (torch.zeros(3, 2, 64).double(), torch.zeros(3, 2, 64).double(), torch.zeros(3, dtype=I32)),
    (torch.zeros(3, 2, 64), torch.zeros(3, 2, 64).half(), torch.zeros(3, dtype=I32)),
    (torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int64)),
    (torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(4, dtype=I32)),
    (torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(6, dtype=I32)[::2]),
])
def test_store_refuses(key, value, slots):
    with pytest.raises(ValueError):
        kv.store_block_kvcache(key, value, *_cache(), slots)


def test_store_refuses_memory_that_is_shared():
    """K and V with one scale tensor, and blocks or heads expanded from one: workgroups would race on them."""
    k, v, ks, vs = _cache()
    rows, slots = torch.zeros(2, 2, 64), torch.zeros(2, dtype=I32)
    for bad in ((k, v, ks, ks), (k[:1].expand(3, -1, -1, -1), v, ks, vs), (k, v[:, :1].expand(-1, 2, -1, -1, -1), ks, vs),
                (k, v, ks[:1].expand(3, -1), vs[:1].expand(3, -1))):
        with pytest.raises(ValueError, match="memory of their own"):
            kv.store_block_kvcache(rows, rows, *bad, slots)


def test_gather_refuses_other_types():
    with pytest.raises(ValueError):
        kv.gather_block_kvcache(*_cache(), torch.zeros(3, dtype=I32), dtype=torch.int8)


def _attend(**change):
    c = _cache()
    a = dict(q=torch.zeros(5, 4, 64, dtype=torch.bfloat16), k_cache=c[0], v_cache=c[1], k_scale=c[2], v_scale=c[3],
             block_tables=torch.zeros((2, 3), dtype=I32), context_lens=torch.zeros(2, dtype=I32),
             cu_seqlens=torch.zeros(3, dtype=I32), max_seqlen=4)
    a.update(change)
    return kv.block_attention(**a)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(5, 4, 64)),
    dict(q=torch.zeros(5, 3, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(5, 0, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(5, 4, 128, dtype=torch.bfloat16)),
    dict(q=torch.zeros(4, 64, dtype=torch.bfloat16)),
    dict(block_tables=torch.zeros((3, 3), dtype=I32)),
    dict(block_tables=torch.zeros((2, 3), dtype=torch.int64)),
    dict(block_tables=torch.zeros((3, 2), dtype=I32).t()),
    dict(block_tables=torch.zeros((0, 3), dtype=I32), context_lens=torch.zeros(0, dtype=I32)),
    dict(context_lens=torch.zeros(2)),
    dict(cu_seqlens=torch.zeros(2, dtype=I32)),
    dict(cu_seqlens=torch.zeros(3, dtype=torch.int64)),
    dict(cu_seqlens=None),
    dict(max_seqlen=0), dict(max_context=-1),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-float("inf")),
    dict(out=torch.zeros(5, 4, 64)),
    dict(out=torch.zeros(4, 4, 64, dtype=torch.bfloat16)),
    dict(out=torch.zeros(5, 64, 4, dtype=torch.bfloat16).transpose(1, 2)),
    dict(out=torch.zeros(5, 4, 66, dtype=torch.bfloat16)[..., :64]),
])
def test_attention_refuses(change):
    with pytest.raises(ValueError):
        _attend(**change)


def test_library_refuses_without_launching():
    """The C entry points on made-up aligned addresses that nothing reads."""
    if not _native.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _native.lib()
    p = [ctypes.c_void_p(i << 12) for i in range(1, 16)]

    def tables(num_seqs=1, width=1, free=1, bs=16, tokens=1, count_out=p[9]):
        return lib.fdms_block_tables(p[0], p[1], num_seqs, p[2], 1, width, p[3], free, p[4], bs, tokens, p[5], p[6],
                                     p[7], p[8], count_out, p[10], None)
    for bad in (dict(num_seqs=0), dict(num_seqs=4097), dict(width=-1), dict(free=-1), dict(bs=48), dict(bs=512),
                dict(tokens=-1), dict(count_out=p[4])):
        assert tables(**bad) == 1, bad

    def store(key=p[0], dtype=_native.DT_BF16, ks_t=128, kc=p[2], kc_b=2048, tokens=1, nb=4, bs=16, h=1, d=64):
        return lib.fdms_store_block_kvcache(key, p[1], dtype, ks_t, 64, 128, 64, kc, p[3], 0, kc_b, 1024, 2048, 1024,
                                            p[4], p[5], 2, p[6], tokens, nb, bs, h, d, None)
    for bad in (dict(key=ctypes.c_void_p(4104)), dict(dtype=3), dict(dtype=-1), dict(ks_t=100), dict(kc_b=8),
                dict(kc=ctypes.c_void_p(4100)), dict(tokens=-1), dict(nb=0), dict(nb=2 ** 27), dict(bs=0),
                dict(bs=17), dict(h=0), dict(d=96)):
        assert store(**bad) == 1, bad
    assert store(tokens=0) == 0

    def gather(out=p[8], dtype=_native.DT_BF16, stride=128, tokens=1, d=64):
        return lib.fdms_gather_block_kvcache(p[2], p[3], 0, 2048, 1024, 2048, 1024, p[4], p[5], 2, p[6], tokens, 4, 16,
                                             1, d, out, p[9], dtype, stride, 64, 128, 64, None)
    for bad in (dict(out=ctypes.c_void_p(4098)), dict(dtype=3), dict(stride=127), dict(tokens=-1), dict(d=32)):
        assert gather(**bad) == 1, bad
    assert gather(tokens=0) == 0

    def attend(q=p[0], dtype=_native.DT_BF16, rows=2, cu=p[7], out=p[8], ws=p[9], seqs=2, h=1, g=4, d=64, nb=4, bs=16,
               most=1, few=1, splits=1, share=4, tiles=0, os_t=256, scale=0.1):
        return lib.fdms_block_attention(q, dtype, 256, 64, rows, p[2], p[3], 0, 1024, 1024, 1024, 1024, p[4], p[5], 1,
                                        p[6], 4, 4, p[10], cu, out, os_t, 64, ws, seqs, h, g, d, nb, bs, most, few,
                                        splits, share, tiles, scale, None)
    for bad in (dict(q=ctypes.c_void_p(4104)), dict(dtype=_native.DT_F32), dict(rows=-1), dict(out=ctypes.c_void_p(4098)),
                dict(splits=0), dict(splits=2, ws=None), dict(splits=-1), dict(splits=257), dict(share=0), dict(seqs=0), dict(h=0), dict(g=0), dict(d=96), dict(nb=0),
                dict(bs=20), dict(most=0), dict(few=-1, tiles=1), dict(few=9), dict(most=2), dict(few=0, splits=0), dict(cu=None, rows=3), dict(cu=None, most=2), dict(os_t=6),
                dict(scale=float("inf")), dict(scale=float("nan"))):
        assert attend(**bad) == 1, bad
    assert attend(rows=0) == 0
