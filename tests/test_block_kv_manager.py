"""The block KV manager's host side: slots, room, and what a step refuses before any launch (CPU)."""
import pytest
import torch

from fastdms_amd.engine.block_kv import BlockKVManager
from fastdms_amd.layers.attention import Attention
from fastdms_amd.utils.context import get_context, reset_context, set_context


def _manager(**change):
    a = dict(num_layers=2, num_kv_heads=1, head_dim=64, num_blocks=6, max_seqs=3, max_model_len=80, block_size=16,
             device="cpu")
    a.update(change)
    return BlockKVManager(**a)


def test_slots_are_given_lowest_first_and_returned():
    m = _manager()
    assert [m.allocate(i) for i in (7, 8, 9)] == [0, 1, 2]
    with pytest.raises(RuntimeError):
        m.allocate(10)
    with pytest.raises(ValueError):
        m.allocate(8)
    m.release(8)
    assert m.allocate(11) == 1 and m.slots == {7: 0, 9: 2, 11: 1}


def test_room_counts_blocks_that_a_step_opens():
    m = _manager()
    m.allocate(1)
    m.allocate(2)
    assert m.can_append({1: 16, 2: 80}) and not m.can_append({1: 17, 2: 80})
    m.cached[0], m.free = 15, 1
    assert m.can_append({1: 1}) and m.can_append({1: 17}) and not m.can_append({1: 18})


def test_release_returns_the_blocks_of_the_sequence():
    m = _manager()
    m.allocate(5)
    m.cached[0], m.free = 33, 3
    m.block_tables[0, :3] = torch.tensor([4, 0, 2], dtype=torch.int32)
    m.release(5)
    assert m.free == 6 and m.free_count.item() == 6
    assert m.free_blocks[3:].tolist() == [4, 0, 2]
    assert (m.block_tables[0] == -1).all() and m.cached[0] == 0


@pytest.mark.parametrize("new,num_tokens,error", [
    ({1: 0}, None, ValueError), ({1: 81}, None, ValueError), ({}, None, ValueError), ({1: 3}, 2, ValueError),
    ({1: 80, 2: 33}, None, RuntimeError), ({4: 1}, None, KeyError),
])
def test_steps_that_do_not_fit_change_nothing(new, num_tokens, error):
    m = _manager()
    m.allocate(1)
    m.allocate(2)
    reset_context()
    with pytest.raises(error):
        m.begin_step(new, num_tokens=num_tokens)
    assert m.free == 6 and m.cached == [0, 0, 0] and get_context().slot_mapping is None


def test_decode_without_any_cache_is_refused():
    attn = Attention(2, 64, 0.1, 1)
    set_context(False)
    try:
        with pytest.raises(RuntimeError, match="compact KV or a block KV cache"):
            attn(torch.zeros(1, 2, 64), torch.zeros(1, 1, 64), torch.zeros(1, 1, 64))
    finally:
        reset_context()


def test_modules_get_their_layers_cache():
    m = _manager()
    mods = [Attention(2, 64, 0.1, 1) for _ in range(2)]
    m.attach_attention_modules(mods)
    assert [x.layer_id for x in mods] == [0, 1]
    assert all(x.block_kv_cache is c for x, c in zip(mods, m.caches))
    with pytest.raises(ValueError):
        m.attach_attention_modules(mods[:1])
