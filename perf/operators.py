"""What the dense 8-bit block KV cache's operators are measured by.

A cache of blocks of `bs` tokens holds each kv head's rows in 8 bits (int8 or
e4m3fn) with one scale per (block, head) for K and one for V:

  K codes  [blocks, heads, bs, D]          k_scale [blocks, heads] fp32
  V codes  [blocks, heads, bs / 16, D, 16] v_scale [blocks, heads] fp32

(V in tiles of 16 tokens, each tile transposed).  Four operators work on it:

  tables   a step's block tables and slot map from the requests' lengths
  store    new K/V rows into their blocks, then the touched blocks' rows read
           back dense, as a compaction of the prompt reads them
  attend   causal attention of the step's queries over the cached rows

`own` False computes them in plain torch, True through the framework.  Widths
are those of the two presets (32 query heads over 8 kv heads, head_dim 64 and
128); block sizes are the compact pages' 16 rows and the engine's default
kvcache_block_size, 256.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
CODES = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0)}
TILE = 16


def listed():
    return [
        # a decode step of a loaded server: 256 sequences, one token each
        dict(name="tables-decode", op="tables", batch=256, cached_lo=1, cached_hi=8192, new_lo=1, new_hi=1, chunk=0,
             bs=16, pad=0, lens=1),
        # a prefill step: 48 ragged prompts, some over an earlier chunk, in a padded batch
        dict(name="tables-prefill", op="tables", batch=48, cached_lo=0, cached_hi=2000, new_lo=1, new_hi=8192, chunk=0,
             bs=16, pad=500, lens=2),
        # a decode step's rows of one layer
        dict(name="store-decode", op="store", dtype="int8", batch=33, cached_lo=1, cached_hi=500, new_lo=1, new_hi=1,
             chunk=0, bs=16, heads=8, dim=128, lens=3),
        # the rows of a prefill batch of 4-8k-token prompts, one layer of the 1B shape
        dict(name="store-prefill-fp8", op="store", dtype="fp8", batch=3, cached_lo=0, cached_hi=700, new_lo=4001,
             new_hi=8192, chunk=0, bs=16, heads=8, dim=64, lens=4),
        # one layer of the 8B shape in 256-token blocks, over earlier chunks that end inside a block
        dict(name="store-prefill-int8", op="store", dtype="int8", batch=5, cached_lo=3, cached_hi=4000, new_lo=200,
             new_hi=8000, chunk=0, bs=256, heads=8, dim=128, lens=5),
        # one user's decode step
        dict(name="attend-1seq", op="attend", dtype="fp8", batch=1, cached_lo=7990, cached_hi=7990, new_lo=1, new_hi=1,
             chunk=0, bs=16, group=4, heads=8, dim=64, lens=6),
        # the benchmark's batch: 8 sequences of 4-8k tokens
        dict(name="attend-8seq", op="attend", dtype="int8", batch=8, cached_lo=4096, cached_hi=8191, new_lo=1,
             new_hi=1, chunk=0, bs=16, group=4, heads=8, dim=128, lens=7),
        # a loaded server: 64 sequences of a few hundred to 32k tokens
        dict(name="attend-64seq", op="attend", dtype="int8", batch=64, cached_lo=300, cached_hi=32000, new_lo=1,
             new_hi=1, chunk=0, bs=16, group=4, heads=8, dim=128, lens=8),
        # a step that checks five drafted tokens a sequence
        dict(name="attend-verify", op="attend", dtype="fp8", batch=16, cached_lo=1000, cached_hi=9000, new_lo=5,
             new_hi=5, chunk=0, bs=256, group=4, heads=8, dim=128, lens=9),
        # a chunk of a long prompt over its earlier chunks
        dict(name="attend-chunk", op="attend", dtype="int8", batch=1, cached_lo=30011, cached_hi=30011, new_lo=777,
             new_hi=777, chunk=0, bs=256, group=4, heads=8, dim=128, lens=10),
        # a prefill batch of ragged prompts
        dict(name="attend-prefill", op="attend", dtype="fp8", batch=4, cached_lo=0, cached_hi=300, new_lo=1500,
             new_hi=6000, chunk=0, bs=16, group=4, heads=8, dim=64, lens=11),
        # decoding sequences with one prompt's chunk among them
        dict(name="attend-mixed", op="attend", dtype="int8", batch=16, cached_lo=500, cached_hi=8000, new_lo=1,
             new_hi=1, chunk=1000, bs=16, group=4, heads=8, dim=128, lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "store", "attend", "attend"])
    case = dict(op=op, lens=rng.randrange(1 << 20), bs=rng.choice([16, 32, 64, 128, 256]), chunk=0)
    if op == "tables":
        if rng.random() < 0.5:
            return case | dict(batch=_log(rng, 1, 512), cached_lo=0, cached_hi=_log(rng, 1, 32768), new_lo=1, new_hi=1,
                               pad=rng.randrange(40))
        return case | dict(batch=_log(rng, 1, 48), cached_lo=0, cached_hi=_log(rng, 1, 2000), new_lo=0,
                           new_hi=_log(rng, 2, 8192), pad=rng.randrange(600))
    case |= dict(dtype=rng.choice(["int8", "fp8"]), dim=rng.choice([64, 128]), heads=rng.choice([1, 2, 4, 8]))
    if op == "store":
        if rng.random() < 0.4:
            return case | dict(batch=_log(rng, 1, 256), cached_lo=0, cached_hi=_log(rng, 1, 500), new_lo=1, new_hi=1)
        return case | dict(batch=rng.randrange(1, 6), cached_lo=0, cached_hi=_log(rng, 1, 4000), new_lo=1,
                           new_hi=_log(rng, 2, 8000))
    case |= dict(group=rng.choice([1, 2, 3, 4, 5, 7, 8]))
    way = rng.random()
    if way < 0.4:
        return case | dict(batch=_log(rng, 1, 64), cached_lo=0, cached_hi=_log(rng, 2, 16000), new_lo=1, new_hi=1)
    if way < 0.6:
        return case | dict(batch=_log(rng, 1, 16), cached_lo=0, cached_hi=_log(rng, 2, 9000), new_lo=1,
                           new_hi=rng.randrange(2, 9))
    if way < 0.8:
        return case | dict(batch=1, cached_lo=0, cached_hi=_log(rng, 1, 30000), new_lo=1, new_hi=_log(rng, 2, 777))
    if way < 0.9:
        return case | dict(batch=rng.randrange(1, 5), cached_lo=0, cached_hi=_log(rng, 1, 300), new_lo=1,
                           new_hi=_log(rng, 2, 4000))
    return case | dict(batch=rng.randrange(2, 13), cached_lo=1, cached_hi=_log(rng, 2, 8000), new_lo=1, new_hi=1,
                       chunk=_log(rng, 2, 1000))


# ---------------------------------------------------------------- lengths
def _lens(case):
    """(cached, new) token counts of the step's sequences; a new count of 0 is a sequence that sits the step out."""
    rng = random.Random(case["lens"])
    cached, new = [], []
    for _ in range(case["batch"]):
        lo, hi = case["cached_lo"], case["cached_hi"]
        cached.append(_log(rng, lo + 1, hi + 1) - 1 if hi > 10 * (lo + 1) else rng.randint(lo, hi))
        new.append(rng.randint(case["new_lo"], case["new_hi"]))
    if case["chunk"]:
        new[0] = case["chunk"]
    if not sum(new):
        new[0] = 1
    return cached, new


def _blocks(n, bs):
    return -(-n // bs)


def work(case):
    cached, new = _lens(case)
    bs = case["bs"]
    t = sum(new)
    if case["op"] == "tables":
        fresh = sum(_blocks(c + n, bs) - _blocks(c, bs) for c, n in zip(cached, new))
        # lengths in; slots (4), positions (8), offsets, context lengths and the new entries out
        return {"bytes": 16 * case["batch"] + 12 * (t + case["pad"]) + 8 * fresh, "flops": t}
    row = case["heads"] * case["dim"]
    if case["op"] == "store":
        rows = sum(c + n - c // bs * bs for c, n in zip(cached, new) if n)  # of the touched blocks
        return {"bytes": row * (2 * t * (2 + 1) + 2 * rows * (1 + 2)), "flops": row * 2 * (t + rows)}
    ctx = sum(c + n for c, n in zip(cached, new) if n)
    seen = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
    blocks = sum(_blocks(c + n, bs) for c, n in zip(cached, new) if n)
    hq = case["heads"] * case["group"]
    return {"bytes": 2 * row * ctx + blocks * (8 * case["heads"] + 4) + 4 * t * hq * case["dim"],
            "flops": 4 * hq * case["dim"] * seen}


# ---------------------------------------------------------------- inputs
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).to(DEV)


def _cu(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _encode(x, dtype):
    """(codes, scales) of blocks x [..., rows, D]: the least power of two whose codes hold the largest value."""
    kind, top = CODES[dtype]
    amax = x.abs().amax(dim=(-1, -2)).double()
    scale = torch.exp2(torch.ceil(torch.log2(amax / top))).float()
    y = x / scale[..., None, None]
    return (y.round() if dtype == "int8" else y).clamp(-top, top).to(kind), scale


def _channels(gen, heads, dim):
    """Channel magnitudes of K: near one another, a few channels of every head far larger."""
    mag = torch.exp(0.4 * torch.randn(heads, 1, dim, generator=gen, device=DEV))
    far = torch.rand(heads, 1, dim, generator=gen, device=DEV) < 0.03
    return torch.where(far, 5.0 * mag, mag)


def _filled(case, gen, blocks):
    """A cache of `blocks` blocks holding earlier rows, made some blocks at a time."""
    h, bs, d = case["heads"], case["bs"], case["dim"]
    kind = CODES[case["dtype"]][0]
    s = dict(k_cache=torch.empty((blocks, h, bs, d), device=DEV, dtype=kind),
             v_cache=torch.empty((blocks, h, bs // TILE, d, TILE), device=DEV, dtype=kind),
             k_scale=torch.empty((blocks, h), device=DEV), v_scale=torch.empty((blocks, h), device=DEV))
    mag = _channels(gen, h, d)
    step = max(1, (1 << 26) // (h * bs * d))
    for b0 in range(0, blocks, step):
        n = min(step, blocks - b0)
        x = torch.randn((n, h, bs, d), generator=gen, device=DEV)
        code, s["k_scale"][b0:b0 + n] = _encode(x * mag, case["dtype"])
        s["k_cache"][b0:b0 + n] = code
        x = torch.randn((n, h, bs, d), generator=gen, device=DEV)
        code, s["v_scale"][b0:b0 + n] = _encode(x, case["dtype"])
        s["v_cache"][b0:b0 + n] = code.view(n, h, bs // TILE, TILE, d).transpose(3, 4)
    return s, mag


def _tables(case, gen, cached, new, spare):
    """Block tables of the sequences over a shuffled pool, and the pool's size."""
    bs = case["bs"]
    need = [_blocks(c + n, bs) for c, n in zip(cached, new)]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, generator=gen, device=DEV).to(torch.int32)
    width = max(need) + 1
    at = torch.full((case["batch"], width), -1, dtype=torch.int64)
    for b, (n, first) in enumerate(zip(need, _cu(need))):
        at[b, :n] = torch.arange(first, first + n)
    at = at.to(DEV)
    return torch.where(at >= 0, order[at.clamp(min=0)], -1).to(torch.int32), order, blocks


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cached, new = _lens(case)
    bs = case["bs"]
    s = dict(op=case["op"], bs=bs, lens=(cached, new), chunk=case["chunk"], max_new=max(new),
             max_context=max(c + n for c, n in zip(cached, new)))
    if case["op"] == "tables":
        held = [_blocks(c, bs) for c in cached]
        table, order, blocks = _tables(case, gen, cached, new, 64)
        col = torch.arange(table.shape[1], device=DEV)
        s["block_tables"] = torch.where(col[None] < _ints(held)[:, None], table, -1)
        # the blocks that no sequence holds, in some order, at the stack's bottom
        taken = torch.zeros(blocks + 1, device=DEV, dtype=torch.bool)
        taken[s["block_tables"].long().flatten()] = True
        taken[blocks] = False
        free = order[~taken[:blocks][order.long()]]
        s["free_blocks"] = torch.cat([free, torch.full((sum(held),), -7, device=DEV, dtype=torch.int32)])
        return s | dict(free_count=_ints([free.numel()]), cached=_ints(cached), new=_ints(new),
                        num_tokens=sum(new) + case["pad"])
    h, d, t = case["heads"], case["dim"], sum(new)
    table, _, blocks = _tables(case, gen, cached, new, 8)
    more, mag = _filled(case, gen, blocks)
    s |= more
    s["block_tables"] = table
    s["dtype"] = case["dtype"]
    if case["op"] == "store":
        hq = 4 * h  # keys and values are views of the qkv projection's rows
        qkv = torch.randn((t, (hq + 2 * h) * d), generator=gen, device=DEV)
        qkv[:, hq * d:(hq + h) * d] *= mag.reshape(1, h * d)
        qkv[:, hq * d:] *= torch.exp(0.3 * torch.randn((t, 1), generator=gen, device=DEV))
        qkv = qkv.to(BF16)
        s["key"] = qkv[:, hq * d:(hq + h) * d].view(t, h, d)
        s["value"] = qkv[:, (hq + h) * d:].view(t, h, d)
        slots, reads = [], []
        tab = table.cpu()
        for b, (c, n) in enumerate(zip(cached, new)):
            if n:
                p = torch.arange(c // bs * bs, c + n)
                slot = tab[b, p // bs] * bs + p % bs
                reads.append(slot)
                slots.append(slot[c % bs:])
        s["slot_mapping"], s["read_slots"] = (_ints(torch.cat(x).tolist()) for x in (slots, reads))
        return s
    hq = h * case["group"]
    q = torch.randn((t, hq, d), generator=gen, device=DEV)
    q /= mag.repeat_interleave(case["group"], 0).reshape(1, hq, d)
    s["q"] = (1.5 * q).to(BF16)
    s["context_lens"] = _ints([c + n for c, n in zip(cached, new)])
    s["cu_seqlens"] = _ints(_cu(new))
    return s


# ---------------------------------------------------------------- the operators
def run(s):
    return {"tables": _run_tables, "store": _run_store, "attend": _run_attend}[s["op"]](s)


def _run_tables(s):
    if own:
        from fastdms_amd.layers.block_kv import prepare_block_tables
        plan = prepare_block_tables(s["cached"], s["new"], s["block_tables"], s["free_blocks"], s["free_count"],
                                    block_size=s["bs"], num_tokens=s["num_tokens"])
        return dict(block_tables=s["block_tables"], slot_mapping=plan.slot_mapping, positions=plan.positions,
                    cu_seqlens=plan.cu_seqlens, context_lens=plan.context_lens, free_count=plan.free_count)
    bs, cached, new, table = s["bs"], s["cached"], s["new"], s["block_tables"]
    ctx = cached + new
    held, need = (cached + bs - 1) // bs, (ctx + bs - 1) // bs
    fresh = need - held
    first = torch.cumsum(fresh, 0) - fresh
    col = torch.arange(table.shape[1], device=DEV)[None]
    at = s["free_count"] - 1 - (first[:, None] + col - held[:, None])
    popped = s["free_blocks"][at.clamp(0, s["free_blocks"].numel() - 1)]
    table = torch.where((col >= held[:, None]) & (col < need[:, None]), popped, table)
    cu = torch.cat([torch.zeros(1, device=DEV, dtype=torch.int64), torch.cumsum(new, 0)])
    t = torch.arange(s["num_tokens"], device=DEV)
    live = t < cu[-1]
    seq = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=new.numel() - 1)
    pos = torch.where(live, cached[seq] + t - cu[seq], 0)
    entry = table[seq, (pos // bs).clamp(max=table.shape[1] - 1)]
    slot = torch.where(live, entry * bs + (pos % bs).to(torch.int32), -1)
    return dict(block_tables=table, slot_mapping=slot.to(torch.int32), positions=pos, cu_seqlens=cu.to(torch.int32),
                context_lens=ctx, free_count=(s["free_count"] - fresh.sum()).to(torch.int32))


def _rows_of(k_codes, v_codes, k_scale, v_scale, bs, slots):
    """Dense K, V [rows, heads, D] fp32 of the cache's rows at `slots`."""
    blk, off = slots.long() // bs, slots.long() % bs
    k = k_codes[blk, :, off].float() * k_scale[blk][..., None]
    v = v_codes[blk, :, off // TILE, :, off % TILE].float() * v_scale[blk][..., None]
    return k, v


def _run_store(s):
    if own:
        from fastdms_amd.layers.block_kv import gather_block_kvcache, store_block_kvcache
        cache = s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
        store_block_kvcache(s["key"], s["value"], *cache, s["slot_mapping"])
        k, v = gather_block_kvcache(*cache, s["read_slots"])
        return dict(k=k, v=v, k_scale=s["k_scale"], v_scale=s["v_scale"])
    bs, (kind, top) = s["bs"], CODES[s["dtype"]]
    blocks, h = s["k_scale"].shape
    d = s["key"].shape[2]
    slot = s["slot_mapping"].long()
    off = torch.full((blocks, bs), bs, device=DEV).view(-1).scatter(0, slot, slot % bs).view(blocks, bs).amin(1)
    touched = off < bs
    before = torch.arange(bs, device=DEV)[None] < off[:, None]  # rows that the block held already
    written = torch.zeros(blocks * bs, device=DEV, dtype=torch.bool).scatter(0, slot, True).view(blocks, bs)
    outs = {}
    for name, rows, codes, old in (("k", s["key"], s["k_cache"], s["k_scale"]),
                                   ("v", s["value"], s["v_cache"].transpose(3, 4).reshape(blocks, h, bs, d),
                                    s["v_scale"])):
        x = torch.zeros((blocks * bs, h, d), device=DEV).index_copy(0, slot, rows.float())
        x = x.view(blocks, bs, h, d).transpose(1, 2)
        amax = x.abs().amax(dim=(-1, -2))
        # the least power of two whose largest code reaches the block's largest new value
        e = torch.floor(torch.log2(amax.double().clamp(min=2.0 ** -126) / top)).clamp(min=-126)
        e = torch.where(torch.exp2(e) * top < amax, e + 1, e)
        need = torch.exp2(e).float()
        scale = torch.where((off > 0)[:, None], torch.maximum(old, need), need)
        scale = torch.where(touched[:, None], scale, old)
        y = torch.where(before[:, None, :, None], codes.float() * (old / scale)[..., None, None],
                        x / scale[..., None, None])
        y = (y.round() if s["dtype"] == "int8" else y).clamp(-top, top).to(kind)
        outs[name] = torch.where((before | written)[:, None, :, None] & touched[:, None, None, None], y.float(),
                                 codes.float())
        outs[name + "_scale"] = scale
    blk, at = s["read_slots"].long() // bs, s["read_slots"].long() % bs
    for name in ("k", "v"):
        outs[name] = (outs[name][blk, :, at] * outs[name + "_scale"][blk][..., None]).to(BF16)
    return outs


def _run_attend(s):
    if own:
        from fastdms_amd.layers.block_kv import block_attention
        return block_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_tables"],
                               s["context_lens"], cu_seqlens=s["cu_seqlens"], max_seqlen=s["max_new"],
                               max_context=s["max_context"])
    if not s["chunk"]:
        return _attend_padded(s, 0, s["max_new"], s["q"])
    # the chunk apart from the decoding sequences, which padding to its length would cost the most
    return torch.cat([_attend_padded(s, 0, s["max_new"], s["q"][:s["max_new"]], 1),
                      _attend_padded(s, 1, 1, s["q"][s["max_new"]:])])


def _attend_padded(s, first, m, q, end=None):
    """Attention of sequences first .. end, their query rows q padded to m a sequence."""
    table, ctx = s["block_tables"][first:end].long().clamp(min=0), s["context_lens"][first:end].long()
    cu = s["cu_seqlens"][first:None if end is None else end + 1].long()
    lo, hi = cu[:-1, None] - cu[0], cu[1:, None] - cu[0]
    t, hq, d = q.shape
    batch, width = table.shape
    h, bs = s["k_cache"].shape[1], s["bs"]
    n = width * bs
    k = (s["k_cache"][table].float() * s["k_scale"][table][..., None, None]).transpose(1, 2).reshape(batch, h, n, d)
    v = s["v_cache"][table].float() * s["v_scale"][table][..., None, None, None]
    v = v.transpose(1, 2).transpose(-1, -2).reshape(batch, h, n, d)
    row = lo + torch.arange(m, device=DEV)[None]
    real = row < hi
    x = torch.where(real[..., None, None], q.float()[row.clamp(max=t - 1)], 0.0)
    x = x.view(batch, m, h, hq // h, d).permute(0, 2, 3, 1, 4).reshape(batch, h, hq // h * m, d)
    p = torch.matmul(x, k.transpose(-1, -2)).view(batch, h, hq // h, m, n) * d ** -0.5
    last = ctx[:, None] - hi + row  # a query's last key
    seen = torch.arange(n, device=DEV)[None, None] <= last[..., None]
    p = p.masked_fill_(~seen[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = torch.matmul(p.view(batch, h, hq // h * m, n), v).view(batch, h, hq // h, m, d)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch * m, hq, d)
    at = torch.where(real, row, t).flatten()
    return torch.zeros((t + 1, hq, d), device=DEV).index_copy(0, at, o)[:t].to(BF16)


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    return (_exact_store if case["op"] == "store" else _exact_attend)(case, s)


def _exact_store(case, s):
    """Block by block of the touched ones, from the definition: scale 2^e with e the least whole number that
    top * 2^e >= max|x| holds for (not under -126), not under an occupied block's; codes to the nearest, ties to
    even; rows already there encoded again from their codes."""
    bs, h, d = case["bs"], case["heads"], case["dim"]
    kind, top = CODES[case["dtype"]]
    slots = s["slot_mapping"].long()
    blk = slots // bs
    order, which = torch.unique(blk, return_inverse=True)
    n = order.numel()
    off = torch.full((n,), bs, device=DEV).scatter_reduce(0, which, slots % bs, "amin")
    result = {}
    for name, rows, codes, old in (("k", s["key"], s["k_cache"][order].to(F64), s["k_scale"][order].to(F64)),
                                   ("v", s["value"], s["v_cache"][order].to(F64).movedim(-1, -2)
                                    .reshape(n, h, bs, d), s["v_scale"][order].to(F64))):
        table = codes * old[:, :, None, None]
        fresh = torch.zeros((n, h, bs, d), device=DEV, dtype=F64)
        fresh[which, :, slots % bs] = rows.to(F64)
        is_new = torch.zeros((n, bs), device=DEV, dtype=torch.bool)
        is_new[which, slots % bs] = True
        amax = fresh.abs().flatten(2).amax(2)
        mant, exp = torch.frexp(amax / top)  # amax / top = mant 2^exp, mant in [0.5, 1)
        e = torch.where(mant == 0.5, exp - 1, exp).to(F64).clamp(min=-126)
        scale = torch.where(amax > 0, torch.exp2(e), torch.full_like(amax, 2.0 ** -126))
        scale = torch.where((off > 0)[:, None], torch.maximum(scale, old), scale)
        keep = torch.arange(bs, device=DEV)[None] < off[:, None]
        x = torch.where(is_new[:, None, :, None], fresh, table) / scale[:, :, None, None]
        if case["dtype"] == "int8":
            y = x.round()
        else:  # three bits after the leading one, the last exponent -6
            step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
            y = (x / step).round() * step
        y = torch.where((keep | is_new)[:, None, :, None], y, codes) * scale[:, :, None, None]
        reads = s["read_slots"].long()
        place = torch.searchsorted(order, reads // bs)
        result[name] = y[place, :, reads % bs]
        full = s[name + "_scale"].to(F64).clone()
        full[order] = scale
        result[name + "_scale"] = full
    return result


def _exact_attend(case, s):
    """One sequence and kv head at a time."""
    cached, new = s["lens"]
    t, hq, d = s["q"].shape
    out = torch.zeros((t, hq, d), device=DEV, dtype=F64)
    g, first = case["group"], 0
    for b, (c, n) in enumerate(zip(cached, new)):
        if n:
            p = torch.arange(c + n, device=DEV)
            slots = s["block_tables"][b].long()[p // case["bs"]] * case["bs"] + p % case["bs"]
            blk, off = slots // case["bs"], slots % case["bs"]
            for h in range(case["heads"]):
                k = s["k_cache"][blk, h, off].to(F64) * s["k_scale"][blk, h, None].to(F64)
                v = s["v_cache"][blk, h, off // TILE, :, off % TILE].to(F64) * s["v_scale"][blk, h, None].to(F64)
                q = s["q"][first:first + n, h * g:(h + 1) * g].to(F64).reshape(n * g, d)
                w = q @ k.T / math.sqrt(d)
                limit = c + torch.arange(n, device=DEV).repeat_interleave(g)
                w = torch.where(p[None] <= limit[:, None], w, -math.inf)
                out[first:first + n, h * g:(h + 1) * g] = (torch.softmax(w, 1) @ v).view(n, g, d)
        first += n
    return out
