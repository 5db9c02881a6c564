"""The memory that an 8-bit cache's kernels read and write lives as long as the cache."""
import gc
import weakref

import torch

from whisperdrz_amd import FlashKVCache8


def test_buffers_outlive_their_attributes():
    cache = FlashKVCache8(2, 40, 1, dtype=torch.float16)
    names = ("k_codes", "v_codes", "k_scales", "v_scales", "k_ring", "v_ring")
    held = {n: (weakref.ref(getattr(cache, n)), getattr(cache, n).data_ptr()) for n in names}
    for n in names:
        setattr(cache, n, getattr(cache, n).clone())
    gc.collect()
    for n, (ref, ptr) in held.items():
        assert ref() is not None and getattr(cache.struct, n) == ptr == ref().data_ptr()
    del cache
    gc.collect()
    assert all(ref() is None for ref, _ in held.values())
