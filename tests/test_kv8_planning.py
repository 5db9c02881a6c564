"""Slots are planned only for 8-bit caches that can be made: heads of 64, 16-bit activations."""
import pytest
import torch

from whisperdrz_amd.kv_cache import FlashKVCache8, KVSlotPool, cache_bytes_per_slot, plan_slots

HUGE = 10**15  # bytes: a pool of a petabyte's slots is refused before anything is allocated


@pytest.mark.parametrize("kw,err", [(dict(head_dim=128), NotImplementedError), (dict(head_dim=32), NotImplementedError),
                                    (dict(dtype=torch.float32), TypeError), (dict(dtype=torch.float8_e4m3fn), TypeError)])
def test_what_8_bit_caches_do_not_hold_is_refused(kw, err):
    with pytest.raises(err):
        plan_slots(272 * 10**9, cache_bits=8, **kw)
    args = dict(n_layers=2, n_heads=20, head_dim=64, self_len=448, cross_len=1500, dtype=torch.bfloat16)
    args.update(kw)
    with pytest.raises(err):
        cache_bytes_per_slot(**args, cache_bits=8)
    with pytest.raises(err):
        KVSlotPool.arena_bytes(3, **args, cache_bits=8)
    with pytest.raises(err):
        KVSlotPool(n_slots=HUGE // (1 << 20), **args, cache_bits=8)
    with pytest.raises(err):
        FlashKVCache8(HUGE // (1 << 20), 1500, 20, args["head_dim"], dtype=args["dtype"])


def test_16_bit_plans_take_any_head_and_type():
    a, b = plan_slots(10**9, n_layers=1, head_dim=64), plan_slots(10**9, n_layers=1, head_dim=128)
    assert b.bytes_per_slot == 2 * a.bytes_per_slot
    assert plan_slots(10**9, n_layers=1, dtype=torch.float32).bytes_per_slot == 2 * a.bytes_per_slot
