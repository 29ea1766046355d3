"""Streams with a window and first positions, as far as the host goes: the plain bookkeeping against the library's own cache,
which pages the cache keeps, the configuration's key, and what is refused before anything is launched."""
import numpy as np
import pytest
import torch

import harness as H  # noqa: F401  (path setup)
import plain_stream as S
from lastengine_b200.cache import Cache, CacheError, StreamCache, StreamStep
from lastengine_b200.parts.base import KVSpec


@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (40, 0), (40, 1), (64, 64), (100, 65), (130, 200), (33, 1000)])
def test_plain_tables_keep_the_pages_that_the_cache_keeps(window, first):
    """The plain bookkeeping and `Cache`, step by step: the same page indexes held, the same number of pages free."""
    cache = Cache({0: KVSpec(1, 8, window=window, first=first)}, max_tokens=64 * 60, max_seqs=4, dtype=torch.float32, device="cpu")
    plain = S.PlainTables(60, 4, 60, 64, window, first)
    rng = np.random.default_rng(3)
    slots = [cache.alloc_seq() for _ in range(3)]
    for step in range(120):
        live = [s for s in slots if rng.random() < 0.8]
        n = [int(rng.integers(1, 90)) if rng.random() < 0.1 else 1 for _ in live]
        t = plain.tables(live, n, sum(n))
        if isinstance(t, int):
            with pytest.raises(Exception):
                cache.reserve(dict(zip(live, n)))
            plain.release(live)
            for s in live:
                cache.free_seq(s)
                assert cache.alloc_seq() == s
            continue
        plain.advance(live, n, t)
        cache.reserve(dict(zip(live, n)))
        cache.commit(dict(zip(live, n)))
        g = cache.kv_groups[0]
        for s in slots:
            assert [p >= 0 for p in g.seq_pages.get(s, [])] == [p >= 0 for p in plain.lists[s]], (step, s)
        assert g.pages.n_free == len(plain.free)
        # everything a next row sees is held
        for s in slots:
            seen = S.sees(torch.tensor([plain.lens[s]]), torch.arange(plain.lens[s]), window, first)[0]
            assert all(plain.lists[s][int(j) // 64] >= 0 for j in torch.nonzero(seen))
        cache.check()


def test_the_key_of_the_configuration_reaches_the_mixer_and_its_cache():
    from lastengine_b200 import ConfigError
    from lastengine_b200.arch.lfm3 import lfm3_plan as build_plan
    from lastengine_b200.config.lfm3 import Lfm3Config
    from lastengine_b200.registry import MIXERS
    from tiny_configs import TINY_C
    plan = build_plan(Lfm3Config.from_dict(dict(TINY_C, sliding_window_first=5)))
    specs = [MIXERS.get(l.mixer.kind)(**l.mixer.params).cache_spec() for l in plan.layers if l.mixer.kind == "attention"]
    assert specs == [KVSpec(5, 48, window=24, first=5), KVSpec(5, 48)]
    plan = build_plan(Lfm3Config.from_dict(TINY_C))
    assert all(l.mixer.params.get("first", 0) == 0 for l in plan.layers)
    with pytest.raises(ConfigError, match="sliding_window_first"):
        Lfm3Config.from_dict(dict(TINY_C, sliding_window_first=-1))


def test_first_positions_without_a_window_change_nothing():
    from lastengine_b200.parts.attention import AttentionMixer
    kw = dict(hidden_size=64, num_heads=4, num_kv_heads=2, head_dim=16, norm_eps=1e-5)
    assert AttentionMixer(first=9, **kw).cache_spec() == KVSpec(2, 16)
    assert AttentionMixer(first=9, chunk=32, **kw).cache_spec() == KVSpec(2, 16, chunk=32, first=9)
    with pytest.raises(ValueError, match="first"):
        AttentionMixer(first=-1, window=3, **kw)


def test_a_stream_cache_says_what_it_does_not_take():
    kw = dict(max_seqs=2, max_tokens=256, max_len=512, device="cpu")
    for bad in (dict(page_size=48), dict(window=-1), dict(first=-2), dict(max_seqs=0)):
        with pytest.raises(ValueError):
            StreamCache(1, 1, 32, **dict(kw, **bad))
    cache = StreamCache(1, 1, 32, window=64, first=4, **kw)
    a, b = cache.open(), cache.open()
    step = cache.plan(2, 3, 2)
    step.set([a, b], [1, 2])
    assert step.slots.tolist() == [a, b] and step.row_counts.tolist() == [1, 2]
    for slots, rows in (([a, a], [1, 2]), ([a], [3]), ([a, b], [1, 1]), ([a, b], [0, 3]), ([a, b], [4, -1])):
        with pytest.raises(CacheError):
            step.set(slots, rows)
    step.set([-1, -1], [1, 2])
    with pytest.raises(CacheError):
        cache.close([a, a])
    with pytest.raises(CacheError):
        cache.close([7])
    assert isinstance(step, StreamStep) and cache.counts.tolist() == [4, 0] and cache.free.tolist() == [3, 2, 1, 0]


def test_calls_off_the_gpu_are_refused():
    from lastengine_b200.ops import kernels as K
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(K.KernelError):
        K.stream_advance(i, i, i, i, i.view(4, 1), i, i[:2], 64)
    with pytest.raises(K.KernelError):
        K.store_rows(torch.zeros(1, 1, 32, 8), torch.zeros(1, 1, 8, 32), torch.zeros(4, 8), torch.zeros(4, 8), i)


def test_a_stream_cache_refuses_lengths_that_32_bits_do_not_count():
    from lastengine_b200.cache import StreamCache
    with pytest.raises(ValueError):
        StreamCache(1, 1, 8, max_seqs=1, max_tokens=64, max_len=2 ** 31, window=64, first=4, device="cpu")
    cache = StreamCache(1, 1, 8, max_seqs=1, max_tokens=64, max_len=128, window=2 ** 40, first=2 ** 40, device="cpu")
    assert cache.kept.tolist() == [2] and (cache.window, cache.first) == (128, 128)
