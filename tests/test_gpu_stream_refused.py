"""Steps of a stream cache that are refused: what their kernels leave, and how the program learns of them."""
import numpy as np
import pytest
import torch

import harness as H  # noqa: F401  (path setup)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def K():
    from lastengine_b200.ops import kernels
    return kernels


def words(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)


def cache_of(**kw):
    from lastengine_b200.cache import StreamCache
    return StreamCache(1, 2, **dict(dict(head_dim=64, max_seqs=3, max_tokens=4 * 64, max_len=512, window=100, first=5, device=DEV), **kw))


def run(cache, slots, counts, nh=4, **kw):
    """One step; its results, where nothing was written NaN."""
    step = cache.plan(len(slots), sum(counts), max(counts))
    step.set(slots, counts)
    cache.begin(step)
    rows = lambda w: torch.randn(sum(counts), w, device=DEV).to(cache.dtype)
    cache.store(0, step, rows(2 * cache.hd), rows(2 * cache.vd))
    out = torch.full((sum(counts), nh * cache.vd), float("nan"), dtype=cache.dtype, device=DEV)
    cache.attend(0, step, out, rows(nh * cache.hd), nh, **kw)
    K().check_device_status()
    return out


@pytest.mark.parametrize("dtype,hd,vd,nh,page,kw", [
    (BF16, 64, 64, 4, 64, {}), (BF16, 128, 128, 4, 64, {}), (BF16, 72, 40, 6, 64, {}), (BF16, 64, 64, 4, 64, {"wide": True}),
    (BF16, 32, 32, 4, 32, {}), (BF16, 96, 96, 2, 32, {"wide": True}), (BF16, 80, 80, 4, 32, {}), (F32, 64, 64, 4, 64, {}), (F32, 33, 7, 8, 32, {})])
@pytest.mark.parametrize("counts", [[1, 1, 1], [200, 1, 90], [3, 0, 120], [0, 300, 0], [40, 40, 41]])
@pytest.mark.parametrize("tiles", [False, True])
def test_the_results_of_a_refused_step_are_zeros(dtype, hd, vd, nh, page, kw, counts, tiles, monkeypatch):
    if tiles:
        monkeypatch.setattr(K(), "STREAM_TILE_WORK", 0)
    cache = cache_of(head_dim=hd, v_head_dim=vd, page_size=page, dtype=dtype)
    slots = [cache.open() for _ in counts]
    kw = dict(kw)
    assert bool(torch.isfinite(run(cache, slots, [64, 64, 65], nh, **kw)).all())      # every page is taken
    k, v, held = cache.k.clone(), cache.v.clone(), cache.lengths(slots)
    while True:      # single tokens are refused once their pages are full
        out = run(cache, slots, counts, nh, **kw)
        if cache.lengths(slots) == held:
            break
        assert max(counts) == 1 and bool(torch.isfinite(out).all())
        k, v, held = cache.k.clone(), cache.v.clone(), cache.lengths(slots)
    assert bool((out == 0).all())
    assert torch.equal(k, cache.k) and torch.equal(v, cache.v)


def test_rows_of_a_refused_step_are_shared_out_or_dropped():
    """Short of pages, longer than the tables, rows that are not as many as the counts say, slots that cannot be; more sequences than rows."""
    for slots, counts, rows, status in (([0, 1, 2], [70, 70, 70], 210, 5), ([0], [200], 200, -1), ([0, 1], [1, 1], 3, -2), ([0, 7], [1, 1], 2, -3),
                                        ([-1] * 9 + [7], [0] * 9 + [4], 4, -3), ([0, 1, -1], [2 ** 31 - 1, 5, 5], 11, -1), ([5], [0], 0, -3)):
        for keep in (False, True):
            lens, kept, pages = words([0] * 3), words([0] * 3), torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
            free, counts2 = words([3, 2, 1, 0]), words([4, 0])
            B = len(slots)
            fill = lambda *s: torch.full(s, -123, dtype=torch.int32, device=DEV)
            table, slot_map, row_seq, row_pos = fill(B, 3), fill(rows), fill(rows), fill(rows)
            slot, qlen, pos0, qstart = (fill(B) for _ in range(4))
            K().stream_tables(table, slot_map, row_seq, row_pos, slot, qlen, pos0, qstart, words(slots), words(counts), lens, pages, free, counts2, 32,
                              keep_rows=keep)
            assert counts2.tolist() == [4, status]
            assert slot.tolist() == [-1] * B and pos0.tolist() == [0] * B and bool((slot_map == -1).all()) and bool((table == -1).all())
            if keep:
                n, at = qlen.tolist(), qstart.tolist()
                assert sum(n) == rows and at == [sum(n[:b]) for b in range(B)] and max(n) - min(n) <= 1
                assert row_seq.tolist() == [b for b in range(B) for _ in range(n[b])]
                assert row_pos.tolist() == [i for b in range(B) for i in range(n[b])]
            else:
                assert qlen.tolist() == [0] * B
            K().stream_advance(slot, qlen, lens, kept, pages, free, counts2, 32)
            assert lens.tolist() == [0] * 3 and counts2.tolist() == [4, status] and free.tolist() == [3, 2, 1, 0] and bool((pages == -1).all())


def test_a_refusal_is_reported_however_many_steps_follow():
    from lastengine_b200.cache import CacheError, CacheFull
    cache = cache_of()
    a, b = cache.open(), cache.open()
    run(cache, [a, b], [64, 128])
    cache.check()
    run(cache, [a, b], [200, 1])                # short of pages
    run(cache, [a, b], [1, 600])                # longer than the tables
    run(cache, [a], [1])
    run(cache, [a], [2])
    with pytest.raises(CacheFull, match="2 steps were refused"):
        cache.check()
    cache.check()                               # reported once
    run(cache, [a], [500])
    run(cache, [a], [1])
    with pytest.raises(CacheError):
        cache.check()
    assert cache.lengths([a, b]) == [68, 128]


def test_replayed_steps_that_were_refused_until_a_sequence_ended_are_reported():
    """A captured decode step is refused while the pages are short, and runs again once another sequence has ended."""
    from lastengine_b200.cache import CacheFull
    cache = cache_of(window=0, first=0)
    a, b = cache.open(), cache.open()
    run(cache, [a, b], [63, 192])
    step = cache.plan(1, 1, 1)
    step.set([a], [1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.begin(step)
    graph.replay()                              # the 64th position
    cache.check()
    for _ in range(5):
        graph.replay()
    cache.close([b])
    for _ in range(3):
        graph.replay()
    assert cache.lengths([a]) == [67]
    with pytest.raises(CacheFull, match="5 steps were refused"):
        cache.check()
    cache.check()


def test_refusals_are_added_up_until_the_program_clears_them():
    lens, pages, free, counts, refused = words([0] * 2), torch.full((2, 2), -1, dtype=torch.int32, device=DEV), words([1, 0]), words([2, 0]), words([0, 0])
    step = lambda slots, n, word=refused: K().stream_tables(torch.zeros(len(n), 2, dtype=torch.int32, device=DEV), *(words([0] * sum(n)) for _ in range(3)),
                                                            *(words([0] * len(n)) for _ in range(4)), words(slots), words(n), lens, pages, free, counts, 32, refused=word)
    step([0], [3])
    assert refused.tolist() == [0, 0] and counts[1] == 0
    step([0, 1], [64, 33])
    step([5], [1])
    step([0], [3])
    assert refused.tolist() == [2, 2] and counts[1] == 0
    refused.copy_(words([2 ** 31 - 1, 7]))
    step([5], [1])
    assert refused.tolist() == [2 ** 31 - 1, 7] and counts[1] == -3
    for bad in (words([0]), refused.long(), refused.cpu()):
        with pytest.raises(K().KernelError):
            step([0], [1], bad)
