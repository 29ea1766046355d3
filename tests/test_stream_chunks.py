"""Which pages `Cache` keeps of layers whose rows see a chunk (or a window within a chunk) and their sequence's first positions."""
import numpy as np
import pytest
import torch

import harness as H  # noqa: F401  (path setup)
from lastengine_b200.cache import Cache
from lastengine_b200.parts.base import KVSpec


@pytest.mark.parametrize("window,chunk,first", [(0, 1, 1), (0, 33, 5), (0, 64, 64), (0, 64, 70), (0, 100, 130), (0, 256, 33), (40, 100, 6), (100, 64, 9), (0, 70, 0)])
def test_the_cache_keeps_what_later_rows_see_and_no_more(window, chunk, first):
    cache = Cache({0: KVSpec(1, 8, window=window, chunk=chunk, first=first)}, max_tokens=64 * 200, max_seqs=2, dtype=torch.float32, device="cpu")
    rng, slot, held = np.random.default_rng(1), cache.alloc_seq(), 0
    for _ in range(150):
        n = int(rng.integers(1, 80)) if rng.random() < 0.2 else 1
        cache.reserve({slot: n})
        cache.commit({slot: n})
        held += n
        pages = cache.kv_groups[0].seq_pages[slot]
        lo = max(held + 1 - window if window else 0, held // chunk * chunk, 0)      # of the next row
        for j, p in enumerate(pages):
            seen = any(t < first or t >= lo for t in range(64 * j, 64 * j + 64))
            assert (p >= 0) == seen, (held, j)
        cache.check()
