"""A model on the dense block KV cache: prompts, a chunk that continues one,
decode steps and a sequence that leaves, through BlockKVManager and the
attention modules, every attention call checked against plain 64-bit code fed
the same q, k, v rows."""
import pytest
import torch

import block_kv_reference as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


class Watch:
    """Runs an attention module and keeps what went in and came out."""

    def __init__(self, module):
        self.module, self.calls = module, []
        self.forward = module.forward
        module.forward = self

    def __call__(self, q, k, v, **kw):
        ins = [x.detach().clone() for x in (q, k, v)]
        out = self.forward(q, k, v, **kw)
        self.calls.append((*ins, out.detach().clone()))
        return out


def _causal(q, k, v, cu, scale):
    """Plain attention of prompts over their own rows, and its bound: P and V
    are bf16 (2^-8 of each weight, the sum of P of the rounded weights as well)."""
    t, hq, d = q.shape
    g = hq // k.shape[1]
    out = torch.zeros((t, hq, d), dtype=torch.float64)
    bound = torch.zeros_like(out)
    q, k, v = (x.cpu().double() for x in (q, k, v))
    for a, b in zip(cu, cu[1:]):
        for i in range(a, b):
            for h in range(hq):
                p = torch.softmax(scale * (k[a:i + 1, h // g] @ q[i, h]), 0)
                o = p @ v[a:i + 1, h // g]
                out[i, h] = o
                err = (p @ v[a:i + 1, h // g].abs()) * (2 * 2.0 ** -8 + 2.0 ** -12)
                bound[i, h] = err + 2.0 ** -8 * (o.abs() + err)
    return out, bound


@pytest.mark.parametrize("name,dtype,block_size", [("tiny-llama", torch.int8, 16),
                                                   ("tiny-qwen3", torch.float8_e4m3fn, 64)])
def test_model_on_blocks(name, dtype, block_size):
    from fastdms_amd.engine.block_kv import BlockKVManager
    from fastdms_amd.models.synthetic import build_synthetic_model, model_config
    cfg = model_config(name)
    model = build_synthetic_model(cfg, seed=3, device=DEV)
    mgr = BlockKVManager(num_layers=cfg.num_hidden_layers, num_kv_heads=cfg.num_key_value_heads,
                         head_dim=cfg.head_dim, num_blocks=40, max_seqs=4, max_model_len=200,
                         block_size=block_size, dtype=dtype, device=DEV)
    modules = [layer.self_attn.attn for layer in model.model.layers]
    mgr.attach_attention_modules(modules)
    watches = [Watch(m) for m in modules]
    caches = [ref.Cache(c) for c in mgr.caches]
    gen = torch.Generator().manual_seed(1)
    for i in range(3):
        mgr.allocate(i)
    steps = [{0: 37, 2: 70}, {1: 9, 2: 1}, {0: 21, 1: 1, 2: 1}, *[{0: 1, 1: 1, 2: 1}] * 4, "leave", {0: 1, 2: 1, 5: 30},
             *[{0: 1, 2: 1, 5: 1}] * 3]
    for new in steps:
        if new == "leave":
            free = mgr.free
            held = -(-mgr.cached[mgr.slots[1]] // block_size)
            mgr.release(1)
            assert mgr.free == free + held
            mgr.allocate(5)
            continue
        before = list(mgr.cached)
        total = sum(new.values())
        step = mgr.begin_step(new, num_tokens=total + 2)
        try:
            ids = torch.randint(0, cfg.vocab_size, (total + 2,), generator=gen).to(DEV)
            with torch.inference_mode():
                hidden = model(ids, step.positions)
            assert torch.isfinite(hidden[:total]).all()
        finally:
            mgr.end_step()
        assert step.status.item() == 0 and step.free_count.item() == mgr.free
        table, slots, cu = mgr.block_tables.tolist(), step.slot_mapping.tolist(), step.cu_seqlens.tolist()
        counts = [b - a for a, b in zip(cu, cu[1:])]
        assert step.positions.tolist()[:total] == [p for c, n in zip(before, counts) for p in range(c, c + n)]
        held = [b for row in table for b in row if b >= 0]
        assert len(held) == len(set(held)) == mgr.num_blocks - mgr.free
        alone = max(counts) > 1 and all(c == 0 or n == 0 for c, n in zip(before, counts))
        for w, c in zip(watches, caches):
            q, k, v, out = w.calls.pop()
            c.store(k, v, slots)
            if alone:
                want, bound = _causal(q[:total], k[:total], v[:total], cu, w.module.scale)
            else:
                want, bound = ref.attention(q[:total], c, table, mgr.cached, cu, w.module.scale)
            assert ((out[:total].cpu().double() - want).abs() <= bound).all(), new
    for c, cache in zip(caches, mgr.caches):
        got = ref.Cache(cache)
        used = sorted(b for row in mgr.block_tables.tolist() for b in row if b >= 0)
        for x in ("k", "v"):
            assert torch.equal(got.scale[x][used], c.scale[x][used])


def test_cached_rows_pack_into_the_compact_layout():
    """A prompt read back from the blocks goes through the compaction as its dense rows would."""
    from fastdms_amd.engine.sequence import Sequence
    from fastdms_amd.engine.paged_kv import PagedCompactKVManager
    from fastdms_amd.layers import block_kv as kv
    from fastdms_amd.sampling_params import SamplingParams
    n, h, d = 90, 2, 64
    cache = kv.allocate_block_kvcache(8, h, 16, d, torch.int8, DEV)
    plan = kv.prepare_block_tables(torch.zeros(1, dtype=torch.int32, device=DEV),
                                   torch.full((1,), n, dtype=torch.int32, device=DEV),
                                   torch.full((1, 8), -1, dtype=torch.int32, device=DEV),
                                   torch.arange(8, dtype=torch.int32, device=DEV),
                                   torch.full((1,), 8, dtype=torch.int32, device=DEV), block_size=16, num_tokens=n)
    g = torch.Generator(device=DEV).manual_seed(4)
    k, v = (torch.randn((n, h, d), generator=g, device=DEV).bfloat16() for _ in range(2))
    kv.store_block_kvcache(k, v, *cache, plan.slot_mapping)
    k2, v2 = kv.gather_block_kvcache(*cache, plan.slot_mapping)
    # each value within half a step of its block's scale
    for x, y, s in ((k, k2, cache[2]), (v, v2, cache[3])):
        step = s[plan.slot_mapping.long() // 16][..., None]
        assert ((x.float() - y.float()).abs() <= 0.5 * step).all()
    evict = torch.rand((n, h), generator=g, device=DEV) < 0.5
    packed = []
    for kk, vv in ((k, v), (k2, v2)):
        mgr = PagedCompactKVManager(num_layers=1, num_kv_heads=h, capacity_tokens=1024, max_model_len=256,
                                    device=torch.device(DEV), head_dim=d, compact_dtype=torch.bfloat16,
                                    max_active_seqs=1)
        seq = Sequence(list(range(n)), SamplingParams(max_tokens=4))
        mgr.allocate(seq)
        mgr.begin_prefill()
        mgr.streaming_pack_layer(layer_id=0, k=kk, v=vv, evict_mask=evict,
                                 cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32, device=DEV),
                                 seq_ids=[seq.seq_id], window_size=16, cu_seqlens_host=[0, n])
        packed.append(mgr.layer_major_live_counts[0, 0].tolist())
    assert packed[0] == packed[1] and 0 < min(packed[0]) < n
