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


def reads(window, chunk, first, pos):
    lo = max(pos + 1 - window if window else 0, pos // chunk * chunk if chunk else 0, 0)
    return {t for t in range(pos + 1) if t >= lo or t < first}


SIGHTS = [(0, 0, 0), (1, 0, 0), (8, 0, 0), (9, 0, 0), (8, 0, 3), (8, 0, 5), (0, 8, 0), (0, 4, 0), (0, 12, 0), (0, 8, 3), (8, 8, 3), (5, 12, 0), (12, 4, 5), (1, 8, 5)]


@pytest.mark.parametrize("owner", SIGHTS)
@pytest.mark.parametrize("reader", SIGHTS)
def test_when_an_entry_holds_what_another_layer_reads(owner, reader):
    """(position by position; a reader without window and chunk sees its first positions anyway)"""
    from lastengine_b200.parts.base import keeps_for
    spec = lambda s: KVSpec(1, 8, window=s[0], chunk=s[1], first=s[2])
    want = all(reads(*reader, pos) <= reads(*owner, pos) for pos in range(100))
    assert keeps_for(spec(owner), spec(reader)) == want


@pytest.mark.parametrize("mine,theirs,fits", [({"window": 32, "first": 4}, {"window": 32, "first": 4}, True), ({"window": 32, "first": 4}, {"window": 32, "first": 70}, False),
                                              ({"window": 32}, {"window": 33}, False), ({"window": 32}, {}, False), ({}, {"window": 32, "first": 9}, True),
                                              ({"window": 64, "first": 9}, {"window": 32, "first": 5}, True)])
def test_a_plan_whose_layer_reads_what_another_layer_s_cache_gave_back_is_refused(mine, theirs, fits):
    import dataclasses
    from lastengine_b200.arch.lfm3 import lfm3_plan
    from lastengine_b200.config import Lfm3Config
    from lastengine_b200.engine.model import Model
    from lastengine_b200.parts.base import BuildEnv, ScheduleEntry
    from tiny_configs import TINY_A
    plan = lfm3_plan(Lfm3Config.from_dict(TINY_A))
    lay = list(plan.layers)
    for i, options in ((1, mine), (3, dict(theirs, own_kv=False))):
        lay[i] = dataclasses.replace(lay[i], mixer=dataclasses.replace(lay[i].mixer, params={**lay[i].mixer.params, **options}))
    plan = dataclasses.replace(plan, layers=lay, schedule=[ScheduleEntry(0), ScheduleEntry(1), ScheduleEntry(2), ScheduleEntry(3, cache=1, writes_cache=False)])
    build = lambda: Model(plan, BuildEnv(torch.device("cpu"), torch.bfloat16))
    if fits:
        build()
    else:
        with pytest.raises(ValueError, match="gives back"):
            build()
