"""The dense 8-bit block KV cache written out plainly, in 64 bits on the CPU
(what the kernels of fastdms_amd.layers.block_kv are compared with)."""
import math

import torch

F64 = torch.float64
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def least_scale(amax: float, top: float) -> float:
    """The least power of two s >= 2^-126 with amax <= top * s."""
    amax = min(amax, torch.finfo(torch.float32).max)
    e = -126
    while top * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def round_codes(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Values / scale in 64 bits -> the nearest code's value (ties to even, saturating)."""
    top = TOP[dtype]
    x = x.clamp(-top, top)
    if dtype == torch.int8:
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-top, top)


class Cache:
    """Codes as values [blocks, heads, block_size, D], scales [blocks, heads]; K and V alike."""

    def __init__(self, tensors):
        k, v, ks, vs = (t.detach().cpu() for t in tensors)
        nb, h, bs, d = k.shape
        self.dtype, self.bs = k.dtype, bs
        self.codes = {"k": k.to(F64), "v": v.to(F64).transpose(3, 4).reshape(nb, h, bs, d)}
        self.scale = {"k": ks.to(F64), "v": vs.to(F64)}

    def store(self, key, value, slots):
        """Runs of consecutive slots of one block, one after another."""
        slots = [int(s) for s in slots]
        nb, h = self.scale["k"].shape
        t = 0
        while t < len(slots):
            s0 = slots[t]
            if s0 < 0 or s0 // self.bs >= nb:
                t += 1
                continue
            n = 1
            while t + n < len(slots) and slots[t + n] == s0 + n and (s0 + n) % self.bs:
                n += 1
            blk, off = divmod(s0, self.bs)
            for name, rows in (("k", key), ("v", value)):
                x = rows[t:t + n].detach().cpu().to(F64)
                x = torch.where(x.isnan(), 0.0, x)
                for j in range(h):
                    s = least_scale(float(x[:, j].abs().max()), TOP[self.dtype])
                    old = float(self.scale[name][blk, j])
                    if off:
                        s = max(s, old)
                        if s > old:
                            c = self.codes[name][blk, j, :off]
                            self.codes[name][blk, j, :off] = round_codes(c * (old / s), self.dtype)
                    self.codes[name][blk, j, off:off + n] = round_codes(x[:, j] / s, self.dtype)
                    self.scale[name][blk, j] = s
            t += n

    def rows(self, name, slots):
        """Dense rows [T, heads, D] of slots (outside the cache: zeros)."""
        slots = torch.as_tensor([int(s) for s in slots], dtype=torch.int64)
        nb = self.scale["k"].shape[0]
        ok = (slots >= 0) & (slots // self.bs < nb)
        blk, off = torch.where(ok, slots, 0) // self.bs, torch.where(ok, slots, 0) % self.bs
        x = self.codes[name][blk, :, off] * self.scale[name][blk][..., None]
        return torch.where(ok[:, None, None], x, 0.0)


def tables(cached, new, table, free, count, bs, num_tokens):
    """prepare_block_tables on lists: (table, slots, positions, cu, context, count)."""
    table = [list(r) for r in table]
    slots, positions, cu = [], [], [0]
    for b, (c, n) in enumerate(zip(cached, new)):
        for at in range(-(-c // bs), -(-(c + n) // bs)):
            count -= 1
            table[b][at] = free[count]
        for p in range(c, c + n):
            slots.append(table[b][p // bs] * bs + p % bs)
            positions.append(p)
        cu.append(cu[-1] + n)
    pad = num_tokens - len(slots)
    return (table, slots + [-1] * pad, positions + [0] * pad, cu, [c + n for c, n in zip(cached, new)], count)


def attention(q, cache: Cache, table, context, cu, scale=None, codes=0.0):
    """(out, bound) [T, Hq, D] in 64 bits.  The bound is what the kernel's
    roundings can add up to, element by element (half a unit in the last place
    is eps / 2 of the value):

    * P is rounded to fp16 relative to its row's largest weight and the largest
      V scale: 2^-11 of itself, or 2^-25 of the row's top below fp16's normal
      range; sums and products of fp32 add a few 2^-24 per term and the scores'
      own error e_s = |s| * (D + 8) * 2^-24 shifts exp(s) by e_s of itself:
      sum_j p_j |v_j| * (2^-11 + 2 e_s + n 2^-24) + n 2^-25 max |v|, over sum p;
    * codes may be held as halves relative to the largest scale of the
      sequence, and then are off by at most 2^-25 of it: e_s grows by scale *
      2^-25 max sK * sum |q|, the result by 2^-25 max sV;
    * scales that are not powers of two: a block's scale over the sequence's
      largest may be rounded to a half and a code's product with it again, each
      2^-11 of itself.  With ``codes`` = 2^-10 + 2^-22 K's part of that is
      codes * |scale| * sum |k q| more in e_s, which is then no longer small
      enough for exp(2 e_s) - 1 = 2 e_s; V's is codes * sum_j p_j |v_j|;
    * the result is rounded once to its type: eps / 2 of itself."""
    t, hq, d = q.shape
    nb, h = cache.scale["k"].shape
    g = hq // h
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros((t, hq, d), dtype=F64)
    bound = torch.zeros((t, hq, d), dtype=F64)
    half = torch.finfo(q.dtype).eps / 2
    q = q.detach().cpu().to(F64)
    for b, ctx in enumerate(context):
        q0, q1 = cu[b], min(cu[b + 1], t)
        if q1 <= q0:
            continue
        ctx = min(ctx, len(table[b]) * cache.bs)
        slots = [table[b][p // cache.bs] * cache.bs + p % cache.bs if 0 <= table[b][p // cache.bs] < nb else -1
                 for p in range(ctx)]
        here = torch.tensor([s >= 0 for s in slots], dtype=torch.bool)
        k, v = cache.rows("k", slots), cache.rows("v", slots)
        blocks = [x for x in table[b][:math.ceil(ctx / cache.bs)] if 0 <= x < nb]
        tops = [[float(cache.scale[x][blocks, j].max()) if blocks else 0.0 for j in range(h)] for x in ("k", "v")]
        for i in range(q1 - q0):
            last = ctx - (q1 - q0) + i
            seen = here & (torch.arange(ctx) <= last)
            n = int(seen.sum())
            if n == 0:
                continue
            kk, vv = k[seen], v[seen]
            for j in range(hq):
                s = scale * (kk[:, j // g] @ q[q0 + i, j])
                p = torch.softmax(s, 0)
                o = p @ vv[:, j // g]
                a = p @ vv[:, j // g].abs()
                es = float(s.abs().max()) * (d + 8) * 2.0 ** -24
                es += abs(scale) * 2.0 ** -25 * tops[0][j // g] * float(q[q0 + i, j].abs().sum())
                shift = 2 * es
                if codes:
                    es += codes * abs(scale) * float((kk[:, j // g].abs() @ q[q0 + i, j].abs()).max())
                    shift = math.expm1(2 * es) + codes
                top = float(p.max())
                out[q0 + i, j] = o
                err = a * (2.0 ** -11 + shift + n * 2.0 ** -24) + top * n * 2.0 ** -25 * float(vv.abs().max())
                err = err + 2.0 ** -25 * tops[1][j // g]
                bound[q0 + i, j] = err + half * (o.abs() + err)
    return out, bound


def cu_of(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def blocks_of(n, bs):
    return math.ceil(n / bs)
