"""The dense 8-bit block KV cache on the GPU against plain 64-bit code:
tables and slot maps (equal), store and read-back (equal bit for bit: powers
of two make every step exact but the one rounding to a code), attention
(within what its roundings add up to, element by element)."""
import random

import pytest
import torch

import block_kv_reference as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
FP8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def _kv():
    from fastdms_amd.layers import block_kv
    return block_kv


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _garbage_cache(nb, h, bs, d, dtype, seed=0):
    """A cache of random bytes (NaN codes of e4m3fn and NaN scales among them)."""
    kv = _kv()
    k, v, ks, vs = kv.allocate_block_kvcache(nb, h, bs, d, dtype, DEV)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for x in (k, v):
        x.view(torch.uint8).copy_(torch.randint(0, 256, x.shape, generator=g, device=DEV, dtype=torch.uint8))
    ks.fill_(float("nan"))
    vs.fill_(float("nan"))
    return k, v, ks, vs


# ---------------------------------------------------------------- tables
@pytest.mark.parametrize("bs", [16, 64, 256])
@pytest.mark.parametrize("cached,new,pad", [
    ([0], [1], 0),
    ([15, 16, 17], [1, 1, 1], 2),
    ([0, 5, 0, 300], [7, 0, 600, 33], 9),
    ([0, 0], [0, 0], 3),
    ([31] * 300, [1] * 300, 20),
    ([i % 40 for i in range(1500)], [i % 7 for i in range(1500)], 100),
])
def test_tables_equal_the_lists(bs, cached, new, pad):
    rng = random.Random(len(cached) + bs)
    n = len(cached)
    width = max(ref.blocks_of(c + m, bs) for c, m in zip(cached, new)) + 2
    total = sum(ref.blocks_of(c + m, bs) for c, m in zip(cached, new))
    ids = list(range(total + 5))
    rng.shuffle(ids)
    table = [[-1] * width for _ in cached]
    for b, c in enumerate(cached):
        for at in range(ref.blocks_of(c, bs)):
            table[b][at] = ids.pop()
    count = len(ids)
    num = sum(new) + pad
    want = ref.tables(cached, new, table, ids, count, bs, num)
    # a table that is a slice of a wider one
    wide = torch.full((n, width + 3), -9, dtype=torch.int32, device=DEV)
    wide[:, 1:1 + width] = _ints(table)
    view = wide[:, 1:1 + width]
    free, cnt = _ints(ids + [-5, -5]), _ints([count])
    for _ in range(2):  # the same step again: nothing it read was changed
        got = _kv().prepare_block_tables(_ints(cached), _ints(new), view, free, cnt, block_size=bs, num_tokens=num)
        assert got.status.item() == 0
        assert view.tolist() == want[0]
        assert got.slot_mapping.tolist() == want[1]
        assert got.positions.tolist() == want[2]
        assert got.cu_seqlens.tolist() == want[3]
        assert got.context_lens.tolist() == want[4]
        assert got.free_count.item() == want[5]
    assert (wide[:, 0] == -9).all() and (wide[:, 1 + width:] == -9).all()
    assert cnt.item() == count and free.tolist() == ids + [-5, -5]


@pytest.mark.parametrize("what", ["blocks", "width", "tokens", "cached", "new", "count", "long"])
def test_tables_that_do_not_fit_change_nothing(what):
    kv = _kv()
    cached, new, bs, width, num, count = [4, 20, 3], [30, 2, 100], 16, 8, 140, 12
    status = 0
    if what == "blocks":
        count, status = 7, kv.STATUS_NO_BLOCKS  # 2 + 0 + 6 are needed
    if what == "width":
        width, status = 6, kv.STATUS_TABLE_WIDTH
    if what == "tokens":
        num, status = 131, kv.STATUS_NUM_TOKENS
    if what == "cached":
        cached[1], status = -1, kv.STATUS_INVALID
    if what == "new":
        new[0], status = -2, kv.STATUS_INVALID
    if what == "count":
        count, status = 13, kv.STATUS_INVALID
    if what == "long":
        cached[2], new[2], status = 2 ** 31 - 1, 1, kv.STATUS_INVALID
    table = torch.full((3, width), 3, dtype=torch.int32, device=DEV)
    before = table.clone()
    got = kv.prepare_block_tables(_ints(cached), _ints(new), table, _ints(list(range(12))), _ints([count]),
                                  block_size=bs, num_tokens=num)
    assert got.status.item() == status
    assert torch.equal(table, before)
    assert (got.slot_mapping == -1).all() and (got.positions == 0).all() and (got.cu_seqlens == 0).all()
    assert got.context_lens.tolist() == [max(c, 0) for c in cached] and got.free_count.item() == count


def test_tables_block_ids_that_make_no_slot():
    """A popped id that is negative, or whose slots pass 31 bits, gives slots of -1."""
    got = _kv().prepare_block_tables(_ints([0, 0, 0]), _ints([3, 2, 1]), torch.zeros((3, 1), dtype=torch.int32,
                                                                                     device=DEV),
                                     _ints([2, 2 ** 30, -4]), _ints([3]), block_size=16, num_tokens=6)
    assert got.status.item() == 0
    assert got.slot_mapping.tolist() == [-1, -1, -1, -1, -1, 32]


# ---------------------------------------------------------------- store and read-back
def _store_case(bs, cached, new, seed=0):
    """Slots of each sequence's new rows and of all rows of its touched blocks, over shuffled blocks."""
    rng = random.Random(seed)
    need = [ref.blocks_of(c + n, bs) for c, n in zip(cached, new)]
    ids = list(range(sum(need) + 3))
    rng.shuffle(ids)
    slots, earlier, reads = [], [], []
    for c, n, k in zip(cached, new, need):
        row = [ids.pop() for _ in range(k)]
        at = [row[p // bs] * bs + p % bs for p in range(c + n)]
        earlier += at[:c]
        slots += at[c:]
        reads += at[c // bs * bs:] if n else []
    return sum(need) + 3, earlier, slots, reads


def _rows(t, h, d, dtype, seed, grow=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((t, h, d), generator=g, device=DEV) * torch.exp2(3 * torch.randn((t, h, 1), generator=g,
                                                                                     device=DEV))
    return (grow * x).to(dtype)


def _same_cache(got, want: ref.Cache):
    """Codes, scales and the rows that nothing wrote, all equal (a NaN code is a NaN)."""
    have = ref.Cache(got)
    for name in ("k", "v"):
        assert torch.equal(have.scale[name].nan_to_num(-1.0), want.scale[name].nan_to_num(-1.0)), name
        assert torch.equal(have.codes[name].nan_to_num(1e9), want.codes[name].nan_to_num(1e9)), name


LENS = [
    ([0], [1]),                       # one token, a new block
    ([0, 0, 0], [16, 15, 17]),
    ([5, 15, 16, 250], [1, 1, 1, 1]),  # a decode step: inside a tile, its last row, a new block
    ([3, 0, 29], [40, 0, 300]),       # blocks that end inside a tile, a sequence with no row
    ([7], [600]),
]


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("lens", LENS)
def test_store_and_gather_equal_the_definition(dtype, d, bs, lens):
    kv, h = _kv(), 3
    cached, new = lens
    nb, earlier, slots, reads = _store_case(bs, cached, new)
    cache = _garbage_cache(nb, h, bs, d, dtype)
    want = ref.Cache(cache)
    for step, (at, grow) in enumerate(((earlier, 0.3), (slots, 1.0))):  # rows already there, then the step's
        k, v = (_rows(len(at), h, d, torch.bfloat16, 10 * step + i, grow) for i in range(2))
        kv.store_block_kvcache(k, v, *cache, _ints(at))
        want.store(k, v, at)
    _same_cache(cache, want)
    for out in (torch.bfloat16, torch.float32, torch.float16):
        gk, gv = kv.gather_block_kvcache(*cache, _ints(reads + [-1, nb * bs]), dtype=out)
        for name, g in (("k", gk), ("v", gv)):
            assert torch.equal(g.cpu(), want.rows(name, reads + [-1, nb * bs]).to(out))


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("bs", [16, 128, 256])
@pytest.mark.parametrize("lens", [
    ([17 * i % 300 for i in range(200)], [1] * 200),                               # many runs of a row
    ([3] * 12 + [0, 250], [2] * 12 + [2000, 700]),                                 # short runs beside long ones
    ([17 * i % 90 for i in range(61)], [1] * 30 + [0] + [40 + i for i in range(30)]),
])
@pytest.mark.parametrize("pad", [0, 2500, 60000])
def test_store_of_many_runs(dtype, bs, lens, pad):
    """Decode rows, short and long runs in one call, with and without padding (a wave looks at 1 to 64 tokens)."""
    kv, h, d = _kv(), 2, 64
    nb, earlier, slots, _ = _store_case(bs, *lens)
    cache = _garbage_cache(nb, h, bs, d, dtype)
    want = ref.Cache(cache)
    for step, (at, grow) in enumerate(((earlier, 0.5), (slots + [-1] * pad, 1.0))):
        k, v = (_rows(len(at), h, d, torch.bfloat16, 10 * step + i, grow) for i in range(2))
        kv.store_block_kvcache(k, v, *cache, _ints(at))
        want.store(k, v, at)
    _same_cache(cache, want)


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("rows", [torch.float32, torch.float16, torch.bfloat16])
def test_store_takes_strided_and_unaligned_rows_and_any_float(dtype, rows):
    kv, h, d, bs = _kv(), 2, 64, 32
    nb, _, slots, _ = _store_case(bs, [0, 0], [37, 70])
    t = len(slots)
    want = None
    for off in (0, 3):  # a view of a wider row, and one off the 16-byte grid
        wide = _rows(t, 1, 3 * h * d + 8, rows, 4)[:, 0]
        k = wide[:, off:off + h * d].view(t, h, d)
        v = wide[:, off + h * d:off + 2 * h * d].view(t, h, d).transpose(1, 2).contiguous().transpose(1, 2)
        cache = _garbage_cache(nb, h, bs, d, dtype)
        want = ref.Cache(cache)
        kv.store_block_kvcache(k, v, *cache, _ints(slots))
        want.store(k, v, slots)
        _same_cache(cache, want)


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
def test_store_of_special_values(dtype):
    """Zeros, subnormals, the largest values, infinities and NaN; a later small row keeps the block's scale."""
    kv, h, d, bs = _kv(), 1, 64, 16
    inf, nan = float("inf"), float("nan")
    rows = torch.zeros((6, 16, 1, d), dtype=torch.float32)
    rows[1, 3, 0, :4] = torch.tensor([1e-45, -1e-38, 2.0 ** -126, 2.0 ** -127])
    rows[2, 15, 0, :3] = torch.tensor([3.4e38, -3.4028235e38, 1.0])
    rows[3, 0, 0, :4] = torch.tensor([inf, -inf, nan, 3e38])
    rows[4, 2, 0, :5] = torch.tensor([nan, 127.0, -127.0, 63.5, 0.5])
    rows[5, 2, 0, :5] = torch.tensor([nan, 448.0, 127.00001, 0.001, -448.0])
    rows = rows.view(96, 1, d).to(DEV)
    slots = list(range(96))
    cache = _garbage_cache(6, h, bs, d, dtype)
    want = ref.Cache(cache)
    kv.store_block_kvcache(rows, -rows, *cache, _ints(slots))
    want.store(rows, -rows, slots)
    _same_cache(cache, want)
    for x in cache[:2]:
        assert not x.float().isnan().any()


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("bs", [16, 256])
def test_store_row_by_row_as_decode_does(dtype, bs):
    """One token a call into two sequences' blocks: scales only rise, earlier codes follow, the rest stays."""
    kv, h, d = _kv(), 2, 128
    cache = _garbage_cache(4, h, bs, d, dtype)
    want = ref.Cache(cache)
    for p in range(40):
        slots = [2 * bs + p % bs if p < bs else 3 * bs + p - bs, p % bs + (p // bs) * bs]
        k, v = _rows(2, h, d, torch.bfloat16, 100 + p), _rows(2, h, d, torch.bfloat16, 200 + p)
        kv.store_block_kvcache(k, v, *cache, _ints(slots))
        want.store(k, v, slots)
        _same_cache(cache, want)


def test_store_skips_slots_outside_the_cache():
    kv, h, d, bs, nb = _kv(), 1, 64, 16, 2
    cache = _garbage_cache(nb, h, bs, d, torch.int8)
    want = ref.Cache(cache)
    slots = [-1, 5, 6, -1, nb * bs, 2 ** 31 - 1, 16, -2 ** 31]
    k, v = _rows(8, h, d, torch.bfloat16, 1), _rows(8, h, d, torch.bfloat16, 2)
    kv.store_block_kvcache(k, v, *cache, _ints(slots))
    want.store(k, v, slots)
    _same_cache(cache, want)


def test_gather_reads_any_slots_in_any_order():
    kv, h, d, bs, nb = _kv(), 2, 128, 32, 5
    cache = kv.allocate_block_kvcache(nb, h, bs, d, FP8, DEV)
    k, v = _rows(nb * bs, h, d, torch.bfloat16, 1), _rows(nb * bs, h, d, torch.bfloat16, 2)
    kv.store_block_kvcache(k, v, *cache, _ints(list(range(nb * bs))))
    want = ref.Cache(cache)
    rng = random.Random(3)
    slots = [rng.randrange(-3, nb * bs + 20) for _ in range(333)]
    gk, gv = kv.gather_block_kvcache(*cache, _ints(slots))
    assert torch.equal(gk.cpu(), want.rows("k", slots).bfloat16())
    assert torch.equal(gv.cpu(), want.rows("v", slots).bfloat16())


# ---------------------------------------------------------------- attention
def _attend_case(bs, h, d, dtype, context, seed=0, spare=2):
    """A cache whose sequences hold `context` rows over shuffled blocks; what no row wrote is random bytes."""
    kv = _kv()
    nb, slots, _, _ = _store_case(bs, context, [0] * len(context), seed)
    rng = random.Random(seed)
    need = [ref.blocks_of(c, bs) for c in context]
    ids = list(range(sum(need) + 3))
    rng.shuffle(ids)
    width = max(need) + spare
    table = []
    for k in need:
        table.append([ids.pop() for _ in range(k)] + [-1] * (width - k))
    cache = _garbage_cache(nb, h, bs, d, dtype, seed)
    if slots:
        k, v = (_rows(len(slots), h, d, torch.bfloat16, seed + 7 + i, 0.25) for i in range(2))
        kv.store_block_kvcache(k, v, *cache, _ints(slots))
    return cache, table


def _check_attention(cache, table, context, lens, group, dtype=torch.bfloat16, seed=0, scale=None, q=None, pad=0,
                     max_context=None, mag=1.0, codes=0.0):
    kv = _kv()
    nb, h, bs, d = cache[0].shape
    cu = ref.cu_of(lens)
    if q is None:
        q = mag * torch.randn((cu[-1] + pad, h * group, d), generator=torch.Generator(device=DEV).manual_seed(seed),
                              device=DEV)
        q = q.to(dtype)
    out = torch.full_like(q, 7.0)
    got = kv.block_attention(q, *cache, _ints(table), _ints(context), cu_seqlens=_ints(cu), max_seqlen=max(lens),
                             max_context=max_context, scale=scale, out=out)
    assert got.data_ptr() == out.data_ptr()
    want, bound = ref.attention(q, ref.Cache(cache), table, context, cu, scale, codes)
    far = (got.cpu().double() - want).abs()[:cu[-1]]
    assert (far <= bound[:cu[-1]]).all(), f"{(far - bound[:cu[-1]]).max()} past the bound, {far.max()} off"
    assert (got[cu[-1]:] == 7.0).all()
    return got


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bs", [16, 32, 256])
@pytest.mark.parametrize("context", [[1], [16, 17], [63, 64, 65, 0], [300, 5, 1025]])
def test_attention_single_tokens(dtype, d, bs, context):
    cache, table = _attend_case(bs, 2, d, dtype, context)
    _check_attention(cache, table, context, [1] * len(context), 4)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 16, 17])
def test_attention_group_sizes(group):
    cache, table = _attend_case(16, 2, 64, torch.int8, [70, 131])
    _check_attention(cache, table, [70, 131], [1, 3], group)


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("context,lens", [
    ([5, 300], [5, 7]),           # a whole short prompt; a few tokens over a context
    ([40, 0, 90], [40, 0, 33]),   # a sequence that sits out, with nothing cached
    ([200, 150], [1, 150]),       # a decoding sequence beside a prompt
    ([257], [130]),
])
def test_attention_query_runs(dtype, d, context, lens):
    cache, table = _attend_case(16, 2, d, dtype, context)
    _check_attention(cache, table, context, lens, 4, pad=5)


def test_attention_queries_that_see_no_key():
    """More queries than keys: the first ones see nothing and get zeros; a context of none gives zeros."""
    cache, table = _attend_case(16, 1, 64, FP8, [3, 0])
    for n in (10, 200):
        got = _check_attention(cache, table, [3, 0], [n, n // 2], 2)
        assert (got[:n - 3] == 0).all() and (got[n:] == 0).all() and (got[n - 3:n] != 0).any()


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("lens", [[2, 3, 1], [50, 45, 20]])
def test_attention_blocks_that_are_not_there(dtype, lens):
    """Entries of -1 or past the cache leave their keys out; contexts past the table's row are cut."""
    cache, table = _attend_case(16, 2, 64, dtype, [100, 90, 64])
    nb = cache[0].shape[0]
    table[0][2], table[1][0], table[1][1] = -1, nb, 2 ** 31 - 1
    table[2] = [-5] * len(table[2])
    got = _check_attention(cache, table, [100, 90, 64], lens, 4)
    assert (got[lens[0] + lens[1]:] == 0).all()
    cut = [r[:4] for r in table]
    _check_attention(cache, cut, [100, 90, 64], lens, 4)


@pytest.mark.parametrize("q_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [None, 0.3, -0.2, 0.0])
@pytest.mark.parametrize("lens", [[1, 4], [3, 50]])
def test_attention_types_and_scales(q_dtype, scale, lens):
    cache, table = _attend_case(32, 2, 128, torch.int8, [77, 200])
    _check_attention(cache, table, [77, 200], lens, 4, dtype=q_dtype, scale=scale)


@pytest.mark.parametrize("n", [6, 42])
def test_attention_large_and_tiny_queries(n):
    """Query magnitudes that a half could not hold, row by row."""
    cache, table = _attend_case(16, 2, 64, FP8, [130])
    q = torch.randn((n, 4, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    q *= torch.tensor([1e30, 1e-30, 1e5, 1e-8, 0.0, 1.0] * (n // 6), device=DEV)[:, None, None]
    q[0] *= 1e-30 / 3e-1
    k = cache[2]
    k *= torch.tensor(2.0 ** -6, device=DEV)  # keep the scores of the large rows moderate
    _check_attention(cache, table, [130], [n], 2, q=q.bfloat16())


@pytest.mark.parametrize("n", [1, 100])
def test_attention_scales_that_differ_widely(n):
    """V scales from 2^-40 to 2^40 in one context: the small blocks' part is lost only below the bound."""
    cache, table = _attend_case(16, 1, 64, torch.int8, [16 * 9])
    cache[3].copy_(torch.exp2(torch.linspace(-40, 40, cache[3].numel(), device=DEV).round()).view_as(cache[3]))
    _check_attention(cache, table, [16 * 9], [n], 4)
    cache[2].copy_(torch.exp2(torch.linspace(-30, -3, cache[2].numel(), device=DEV).round()).view_as(cache[2]))
    _check_attention(cache, table, [16 * 9], [n], 4)


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 7, 60])
def test_attention_scales_that_are_no_powers_of_two(dtype, d, n):
    """Exact for few rows, rounded to halves relative to the largest for many (the bound's codes)."""
    context = [16 * 9 + 5, 200]
    cache, table = _attend_case(32, 2, d, dtype, context)
    g = torch.Generator(device=DEV).manual_seed(5)
    for x in cache[2:]:
        x *= 1 + torch.rand(x.shape, generator=g, device=DEV)
    _check_attention(cache, table, context, [n, n], 4, mag=0.25, codes=2.0 ** -10 + 2.0 ** -22 if n > 8 else 0.0)


@pytest.mark.parametrize("n", [4, 36])
def test_attention_row_of_nan_or_infinite_query_leaves_the_others(n):
    cache, table = _attend_case(16, 1, 64, torch.int8, [50])
    q = torch.randn((n, 2, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).bfloat16()
    clean = _check_attention(cache, table, [50], [n], 2, q=q)
    bad = q.clone()
    bad[n - 3, 0, 5] = float("nan")
    bad[n - 2, 1, 7] = float("inf")
    got = _kv().block_attention(bad, *cache, _ints(table), _ints([50]), cu_seqlens=_ints([0, n]), max_seqlen=n)
    assert got[n - 3, 0].isnan().all() and not got[n - 2, 1].isfinite().all()
    same = torch.ones((n, 2), dtype=torch.bool)
    same[n - 3, 0] = same[n - 2, 1] = False
    assert torch.equal(got.cpu()[same], clean.cpu()[same])


@pytest.mark.parametrize("lens", [[1, 1], [6, 3], [2, 40], [70, 3]])
def test_attention_long_context_splits(lens):
    """Contexts that many workgroups share, one far shorter than the other."""
    context = [9001, 40]
    cache, table = _attend_case(64, 1, 128, torch.int8, context)
    _check_attention(cache, table, context, lens, 4)
    _check_attention(cache, table, context, lens, 4, max_context=9001)


def test_attention_strided_operands():
    """q a view of the projection's rows, out a view, the cache a slice of a layered one, a wide table."""
    kv = _kv()
    context, lens = [90, 33], [2, 1]
    cache, table = _attend_case(16, 2, 64, FP8, context)
    layered = [torch.zeros((x.shape[0], 3, *x.shape[1:]), device=DEV, dtype=x.dtype) for x in cache]
    for big, x in zip(layered, cache):
        big[:, 1].copy_(x)
    views = [big[:, 1] for big in layered]
    wide = torch.full((2, len(table[0]) + 9), 0, dtype=torch.int32, device=DEV)
    wide[:, 4:4 + len(table[0])] = _ints(table)
    qkv = torch.randn((3, 1000), device=DEV).bfloat16()
    q = qkv[:, 8:8 + 8 * 64].view(3, 8, 64)
    out = torch.zeros((3, 8, 100), device=DEV, dtype=torch.bfloat16)
    got = kv.block_attention(q, *views, wide[:, 4:4 + len(table[0])], _ints(context), cu_seqlens=_ints([0, 2, 3]),
                             max_seqlen=2, out=out[:, :, 4:68])
    want, bound = ref.attention(q, ref.Cache(cache), table, context, [0, 2, 3])
    assert ((got.cpu().double() - want).abs() <= bound).all()
    assert (out[:, :, :4] == 0).all() and (out[:, :, 68:] == 0).all()
    odd = qkv[:, 3:3 + 8 * 64].view(3, 8, 64)  # off the 16-byte grid: read through a copy
    got = kv.block_attention(odd, *views, _ints(table), _ints(context), cu_seqlens=_ints([0, 2, 3]), max_seqlen=2)
    want, bound = ref.attention(odd, ref.Cache(cache), table, context, [0, 2, 3])
    assert ((got.cpu().double() - want).abs() <= bound).all()


def test_attention_without_cu_seqlens_is_one_query_each():
    context = [40, 7, 200]
    cache, table = _attend_case(16, 2, 128, torch.int8, context)
    q = torch.randn((3, 8, 128), device=DEV).half()
    kv = _kv()
    a = kv.block_attention(q, *cache, _ints(table), _ints(context))
    b = kv.block_attention(q, *cache, _ints(table), _ints(context), cu_seqlens=_ints([0, 1, 2, 3]), max_seqlen=1)
    assert torch.equal(a, b)


# ---------------------------------------------------------------- as they are used
@pytest.mark.parametrize("dtype", [torch.int8, FP8])
def test_a_run_of_steps(dtype):
    """Two prompts, a chunk that continues one, then decode steps: tables, store and attention in turn."""
    kv, h, g, d, bs, nb = _kv(), 2, 4, 64, 16, 40
    cache = _garbage_cache(nb, h, bs, d, dtype)
    want = ref.Cache(cache)
    table = torch.full((2, 20), -1, dtype=torch.int32, device=DEV)
    free, count = _ints(list(range(nb))), _ints([nb])
    cached, gen = [0, 0], torch.Generator(device=DEV).manual_seed(5)
    host = [[-1] * 20 for _ in range(2)]
    left = nb
    for new in ([37, 60], [0, 90], *([[1, 1]] * 20)):
        t = sum(new)
        plan = kv.prepare_block_tables(_ints(cached), _ints(new), table, free, count, block_size=bs, num_tokens=t)
        host, slots, _, cu, context, left = ref.tables(cached, new, host, list(range(nb)), left, bs, t)
        assert plan.slot_mapping.tolist() == slots and table.tolist() == host
        count = plan.free_count
        qkv = torch.randn((t, (g * h + 2 * h) * d), generator=gen, device=DEV).bfloat16()
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([g * h * d, h * d, h * d], 1))
        kv.store_block_kvcache(k, v, *cache, plan.slot_mapping)
        want.store(k, v, slots)
        got = kv.block_attention(q, *cache, table, plan.context_lens, cu_seqlens=plan.cu_seqlens,
                                 max_seqlen=max(new))
        out, bound = ref.attention(q, want, host, context, cu)
        assert ((got.cpu().double() - out).abs() <= bound).all()
        cached = context
    _same_cache(cache, want)


def test_a_captured_decode_step_replays():
    """Tables, store and attention captured once and replayed over changing inputs, with eager calls between;
    a second graph of the same shapes beside it on another stream."""
    kv, h, g, d, bs, nb = _kv(), 2, 4, 64, 16, 64

    def step(s):
        s["plan"] = kv.prepare_block_tables(s["cached"], s["new"], s["table"], s["free"], s["count"],
                                            block_size=bs, num_tokens=3, out=s.get("plan"))
        kv.store_block_kvcache(s["k"], s["v"], *s["cache"], s["plan"].slot_mapping)
        s["out"] = kv.block_attention(s["q"], *s["cache"], s["table"], s["plan"].context_lens,
                                      cu_seqlens=s["plan"].cu_seqlens, max_seqlen=1, max_context=2000)
        s["count"].copy_(s["plan"].free_count)
        s["cached"].copy_(s["plan"].context_lens)

    def state(seed):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        s = dict(cached=_ints([0, 0]), new=_ints([1, 1]), table=torch.full((2, 125), -1, dtype=torch.int32, device=DEV),
                 free=_ints(list(range(nb))), count=_ints([nb]), cache=_garbage_cache(nb, h, bs, d, torch.int8, seed))
        for name, heads in (("q", h * g), ("k", h), ("v", h)):
            s[name] = torch.randn((3, heads, d), generator=gen, device=DEV).bfloat16()
        return s

    def clone(s):
        return {k: (tuple(x.clone() for x in v) if k == "cache" else v.clone()) for k, v in s.items()
                if k not in ("plan", "out")}

    sides = []
    for seed in (1, 2):
        s = state(seed)
        step(s)  # warm up (and one step into the sequences)
        eager = clone(s)
        graph = torch.cuda.CUDAGraph()
        held = clone(s)
        held["plan"] = kv.BlockTables(*(x.clone() for x in s["plan"]))
        with torch.cuda.graph(graph):
            step(held)
        for k in ("cached", "table", "count"):
            held[k].copy_(eager[k])
        for a, b in zip(held["cache"], eager["cache"]):
            a.copy_(b)
        sides.append((graph, held, eager, torch.cuda.Stream()))
    for i in range(20):
        gen = torch.Generator(device=DEV).manual_seed(100 + i)
        for graph, held, eager, stream in sides:
            for name in ("q", "k", "v"):
                x = torch.randn(held[name].shape, generator=gen, device=DEV).bfloat16()
                held[name].copy_(x)
                eager[name].copy_(x)
        torch.cuda.synchronize()
        for graph, held, eager, stream in sides:
            with torch.cuda.stream(stream):
                graph.replay()
        for graph, held, eager, stream in sides:
            step(eager)
        torch.cuda.synchronize()
        for graph, held, eager, stream in sides:
            assert torch.equal(held["out"][:2], eager["out"][:2]), i
            assert torch.equal(held["table"], eager["table"]) and torch.equal(held["cached"], eager["cached"])
            for a, b in zip(held["cache"][:2], eager["cache"][:2]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_calls_on_two_streams_at_once():
    context = [3000, 2000]
    cache, table = _attend_case(16, 2, 64, torch.int8, context)
    kv = _kv()
    table, ctx = _ints(table), _ints(context)
    qs = [torch.randn((2, 8, 64), device=DEV).bfloat16() for _ in range(2)]
    want = [kv.block_attention(q, *cache, table, ctx) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for q, st in zip(qs, streams):
            with torch.cuda.stream(st):
                got.append(kv.block_attention(q, *cache, table, ctx))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_results_repeat_bit_for_bit():
    context, lens = [5000, 800, 33], [4, 1, 33]
    cache, table = _attend_case(16, 2, 128, FP8, context)
    kv = _kv()
    q = torch.randn((38, 8, 128), device=DEV).bfloat16()
    run = lambda: kv.block_attention(q, *cache, _ints(table), _ints(context), cu_seqlens=_ints(ref.cu_of(lens)),  # noqa
                                     max_seqlen=33)
    first = run()
    for _ in range(5):
        assert torch.equal(run(), first)
