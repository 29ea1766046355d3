"""Streams with a window and first positions that stay visible: attention, the tables built on the device, stores by slot map, and
what runs them together, against plain arithmetic in double precision and plain bookkeeping."""
import math
import types

import numpy as np
import pytest
import torch

import harness as H
import plain_lfm3 as P
import plain_stream as S
from tiny_configs import TINY_C, TINY_D

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def K():
    from lastengine_b200.ops import kernels
    return kernels


def words(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)


# ---- attention -----------------------------------------------------------------------------------------------------
class Case:
    """Sequences of (positions held, rows brought) with their caches: only positions that a row of the step sees are filled, all
    else (also between the first positions and the window) holds NaN; pages that an earlier step would have given back are -1."""

    def __init__(self, seqs, nh, nkv, hd, vd, page, window, first, dtype, seed=0, padding=(), base_page=0, spread=1.0):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.nh, self.nkv, self.hd, self.vd, self.page, self.window, self.first, self.dtype = nh, nkv, hd, vd, page, window, first, dtype
        self.seqs, self.padding = seqs, set(padding)
        self.scale = hd ** -0.5
        lists, n_pages = S.random_lists(rng, [h + n for h, n in seqs], page)
        n_pages += base_page
        lists = [[p + base_page for p in l] for l in lists]
        self.k_pool = torch.full((n_pages, nkv, page, hd), float("nan"), dtype=dtype, device=DEV)
        self.v_pool = torch.full((n_pages, nkv, vd, page), float("nan"), dtype=dtype, device=DEV)
        self.q, self.kv = [], []
        for b, ((h, n), l) in enumerate(zip(seqs, lists)):
            q = (spread * torch.randn(n, nh, hd, generator=g)).to(dtype)
            k, v = torch.randn(h + n, nkv, hd, generator=g).to(dtype), torch.randn(h + n, nkv, vd, generator=g).to(dtype)
            self.q.append(q)
            self.kv.append((k, v))
            if b in self.padding:
                continue
            seen = S.sees(torch.arange(h, h + n), torch.arange(h + n), window, first).any(0)
            for j, p in enumerate(l):
                t = [t for t in range(j * page, min((j + 1) * page, h + n)) if n and seen[t]]
                if t:
                    at = torch.tensor(t)
                    self.k_pool[p, :, at % page] = k[at].permute(1, 0, 2).to(DEV)
                    self.v_pool[p, :, :, at % page] = v[at].permute(1, 2, 0).to(DEV)
            if window > 0:
                for j in range(-(-first // page), max(0, h + 1 - window) // page):
                    l[j] = -1
        pos0 = [0 if b in self.padding else h for b, (h, n) in enumerate(seqs)]
        qlen = [n for h, n in seqs]
        start = np.concatenate([[0], np.cumsum(qlen)[:-1]]) if seqs else []
        self.rows = sum(qlen)
        self.table = torch.from_numpy(S.as_table(lists, max(len(l) for l in lists))).to(DEV)
        self.batch = types.SimpleNamespace(
            n_rows=self.rows, n_seqs=len(seqs), max_qlen=max(qlen), max_kvlen=max(h + n for h, n in seqs),
            row_seq=words(np.repeat(np.arange(len(seqs)), qlen)), row_pos=words(np.concatenate([p + np.arange(n) for p, n in zip(pos0, qlen)])),
            seq_slot=words([-1 if b in self.padding else b for b in range(len(seqs))]), seq_pos0=words(pos0), seq_qstart=words(start),
            seq_qlen=words(qlen))
        self.qd = torch.cat(self.q).reshape(self.rows, nh * hd).to(DEV)

    def run(self, n_splits=None, **kw):
        out = torch.full((self.rows, self.nh * self.vd), float("nan"), dtype=self.dtype, device=DEV)
        general = self.dtype == F32 or self.vd != self.hd
        n = K().attention_splits(self.batch, self.nkv, self.nh // self.nkv, hd=self.hd, window=self.window, general=general, first=self.first) \
            if n_splits is None else n_splits
        scratch = torch.full((self.rows * self.nh * n * (max(self.hd, self.vd) + 2),), float("nan"), device=DEV) if n > 1 else None
        K().attention(out, self.qd, self.k_pool, self.v_pool, self.table, self.batch, self.nh, self.nkv, self.hd, self.page, self.window,
                      self.scale, n_splits=n, scratch=scratch, vd=self.vd, first=self.first, **kw)
        return out

    def check(self, out, slopes=None, sinks=None, factor=None):
        """Roundings, each at its worst: bfloat16 weights and results 2^-8 of what they are (8 significant bits); a score's sum over the head 2^-22 (float32:
        2^-24) of its terms' magnitudes per term, which moves a weight by as much; sums over positions 2^-24 a term; exponentials 2^-20."""
        out = out.double().cpu().view(self.rows, self.nh, self.vd)
        K().check_device_status()
        row = 0
        for b, (h, n) in enumerate(self.seqs):
            got = out[row:row + n]
            row += n
            if b in self.padding:
                assert bool((got == 0).all())
                continue
            if n == 0:
                continue
            k, v = self.kv[b]
            want, mass, size = S.attention(self.q[b].double(), k.double(), v.double(), torch.arange(h, h + n), self.window, self.first,
                                           self.scale, slopes, sinks)
            if factor is not None:
                f = factor[row - n:row]
                want, mass = want * f, mass * f
            T = min(h + n, (self.window or h + n) + self.first)
            if slopes is not None:
                size = size + slopes.abs().max() * (h + n) * 2 ** -4      # the slope's own product and sum
            if self.dtype == BF16:
                bound = 2 ** -8 * (1 + 2 ** -6) * (want.abs() + mass) + 2 * mass * (self.hd * 2 ** -22 * size + T * 2 ** -24 + 2 ** -18)
            else:
                bound = want.abs() * 2 ** -22 + 2 * mass * ((self.hd + 8) * 2 ** -24 * size + T * 2 ** -24 + 2 ** -20)
            off = (got - want).abs()
            assert bool((off <= bound + 1e-30).all()), (b, h, n, float((off / (bound + 1e-30)).nan_to_num(1e9).max()))


WINDOWS = [(1, 1), (17, 1), (64, 64), (40, 70), (100, 4), (130, 129), (300, 33), (33, 1000), (5, 31)]
DECODE = [(0, 1), (1, 1), (31, 1), (63, 1), (64, 1), (65, 1), (127, 1), (200, 1), (511, 1), (700, 1), (1023, 1)]
CHUNKS = [(0, 1), (0, 70), (63, 2), (200, 130), (517, 33), (64, 64), (3, 300)]


@pytest.mark.parametrize("dtype,nh,nkv,hd,vd,page", [
    (BF16, 8, 2, 64, 64, 64), (BF16, 32, 8, 64, 64, 64), (BF16, 3, 1, 32, 32, 32), (BF16, 16, 1, 128, 128, 64), (BF16, 6, 6, 96, 96, 128),
    (BF16, 4, 2, 80, 80, 64), (BF16, 4, 2, 64, 48, 64), (BF16, 5, 5, 20, 12, 32), (BF16, 6, 2, 33, 65, 64), (BF16, 3, 1, 192, 192, 64),
    (BF16, 34, 2, 64, 64, 64), (BF16, 4, 1, 256, 256, 128), (F32, 4, 2, 64, 64, 64), (F32, 6, 2, 80, 48, 32), (F32, 20, 1, 33, 33, 64),
    (F32, 3, 3, 128, 128, 64), (F32, 8, 1, 128, 40, 32), (F32, 5, 1, 256, 200, 64), (F32, 2, 2, 200, 256, 64), (F32, 7, 1, 3, 1, 32)])
@pytest.mark.parametrize("window,first", WINDOWS)
def test_single_tokens(dtype, nh, nkv, hd, vd, page, window, first):
    c = Case(DECODE, nh, nkv, hd, vd, page, window, first, dtype, seed=window + first, padding=[4])
    a = c.run()
    c.check(a)
    for n in (2, 5):
        c.check(c.run(n_splits=n))
    try:
        for n in (1, 2, 3, 8):
            K().set_stream_attention_splits(n)
            c.check(c.run(n_splits=1))
    finally:
        K().set_stream_attention_splits(0)
    assert torch.equal(a, c.run())


@pytest.mark.parametrize("dtype,nh,nkv,hd,vd,page", [
    (BF16, 8, 2, 64, 64, 64), (BF16, 3, 3, 64, 64, 64), (BF16, 8, 1, 64, 64, 64), (BF16, 4, 2, 64, 64, 64), (BF16, 3, 1, 64, 64, 64),
    (BF16, 4, 2, 32, 32, 32), (BF16, 8, 2, 128, 128, 64), (BF16, 3, 3, 128, 128, 64), (BF16, 8, 1, 128, 128, 64), (BF16, 5, 1, 128, 128, 64),
    (BF16, 2, 2, 96, 96, 64), (BF16, 16, 1, 64, 64, 64), (BF16, 2, 1, 64, 64, 128), (BF16, 4, 2, 80, 80, 64), (BF16, 2, 1, 64, 32, 64),
    (BF16, 4, 2, 128, 128, 128),
    (BF16, 2, 1, 8, 128, 192), (BF16, 3, 1, 72, 40, 64), (BF16, 4, 4, 32, 96, 64), (BF16, 2, 1, 64, 20, 64), (BF16, 34, 2, 64, 64, 64),
    (BF16, 2, 1, 192, 192, 64), (F32, 4, 2, 64, 64, 64), (F32, 6, 2, 80, 48, 32)])
@pytest.mark.parametrize("window,first", WINDOWS)
def test_chunks_of_tokens(dtype, nh, nkv, hd, vd, page, window, first):
    c = Case(CHUNKS, nh, nkv, hd, vd, page, window, first, dtype, seed=window + first, padding=[5])
    a = c.run()
    c.check(a)
    assert torch.equal(a, c.run())


@pytest.mark.parametrize("nh,nkv,hd,vd", [(8, 2, 64, 64), (3, 3, 64, 64), (8, 2, 128, 128), (5, 1, 128, 128), (4, 2, 72, 40)])
@pytest.mark.parametrize("window,first", [(1, 1), (64, 64), (300, 33), (33, 1000), (900, 4)])
def test_blocks_that_share_a_tile_s_keys(nh, nkv, hd, vd, window, first):
    """1 to 8 blocks for the keys of a tile, also where some of them get none; with sinks and gates, which the join takes."""
    c = Case(CHUNKS + [(1500, 20), (0, 3)], nh, nkv, hd, vd, 64, window, first, BF16, seed=window, padding=[5])
    g = torch.Generator().manual_seed(1)
    sinks, gate = torch.randn(nh, generator=g), torch.randn(c.rows, nh, generator=g).to(BF16)
    numbers = torch.randn(c.rows, nh * vd, generator=g).to(BF16)
    try:
        for n in (1, 2, 3, 5, 8):
            K().set_stream_attention_splits(n)
            a = c.run()
            c.check(a)
            assert torch.equal(a, c.run())
            c.check(c.run(sinks=sinks.to(DEV), gate=gate.to(DEV)), sinks=sinks.double(), factor=torch.sigmoid(gate.double())[:, :, None])
            c.check(c.run(gate=numbers.to(DEV)), factor=torch.sigmoid(numbers.double()).view(c.rows, nh, vd))
    finally:
        K().set_stream_attention_splits(0)


@pytest.mark.parametrize("seqs", [DECODE, CHUNKS])
def test_weights_of_two_terms_beside_first_positions(seqs):
    """Nearer to the 64-bit result than weights of one term: 2^-16 of a weight where that is 2^-8, but for the rounding of the result."""
    for hd in (64, 128, 32):
        c = Case(seqs, 4, 2, hd, hd, 64, 70, 40, BF16, seed=11)
        wide = c.run(wide=True)
        c.check(wide)
        out, row = wide.double().cpu().view(c.rows, 4, hd), 0
        for (h, n), q, (k, v) in zip(c.seqs, c.q, c.kv):
            want, mass, size = S.attention(q.double(), k.double(), v.double(), torch.arange(h, h + n), 70, 40, c.scale)
            bound = 2 ** -8 * (1 + 2 ** -6) * want.abs() + 2 * mass * (2 ** -16 + hd * 2 ** -22 * size + 110 * 2 ** -24 + 2 ** -18)
            assert bool(((out[row:row + n] - want).abs() <= bound).all()), (hd, h, n)
            row += n


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (4, 4, 32)])
def test_chunks_of_a_few_rows_and_of_none(nh, nkv, hd):
    for seqs in ([(100, 3), (0, 2), (700, 1)], [(100, 0), (5, 9), (300, 0), (64, 64)], [(129, 0), (64, 1), (500, 1)]):
        c = Case(seqs, nh, nkv, hd, hd, 64, 90, 6, BF16)
        c.check(c.run())


@pytest.mark.parametrize("n_seqs", [2, 31, 33, 128, 129, 200])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_sequences_of_unequal_lengths(n_seqs, hd):
    """Tiles are listed for up to 128 sequences of unequal lengths, some of which bring nothing, padding at both ends."""
    rng = np.random.default_rng(n_seqs)
    seqs = [(int(rng.integers(0, 150)), int(rng.integers(0, 7)) if i % 9 else int(rng.integers(40, 120))) for i in range(n_seqs)]
    c = Case(seqs, 4, 2, hd, hd, 64, 60, 5, BF16, seed=n_seqs, padding=[0, n_seqs - 1] if n_seqs > 2 else [])
    c.check(c.run())


@pytest.mark.parametrize("nh,nkv,hd,window,first", [(8, 2, 64, 200, 70), (4, 4, 128, 333, 4), (2, 1, 128, 64, 65), (8, 1, 64, 1, 1)])
def test_many_tiles(nh, nkv, hd, window, first):
    """More tiles than the SMs take at once, and long sequences."""
    c = Case([(0, 1900), (1500, 1301), (77, 800)], nh, nkv, hd, hd, 64, window, first, BF16, seed=5)
    c.check(c.run())


@pytest.mark.parametrize("seqs", [DECODE, CHUNKS])
@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 128), (BF16, 32), (F32, 48)])
def test_slopes_sinks_and_gates_beside_first_positions(seqs, dtype, hd):
    nh, nkv = 4, 2
    c = Case(seqs, nh, nkv, hd, hd, 64, 50, 70, dtype, seed=9)
    g = torch.Generator().manual_seed(1)
    slopes, sinks = 2.0 ** -torch.arange(1, nh + 1).float(), torch.randn(nh, generator=g)
    c.check(c.run(slopes=slopes.to(DEV), sinks=sinks.to(DEV)), slopes.double(), sinks.double())
    gate = torch.randn(c.rows, nh, generator=g).to(dtype)
    c.check(c.run(gate=gate.to(DEV)), factor=torch.sigmoid(gate.double())[:, :, None])


def test_steps_that_only_the_general_kernel_takes():
    """Pools off a 16-byte boundary."""
    for seqs in (DECODE, CHUNKS):
        for dtype, hd, vd in ((F32, 48, 48), (BF16, 72, 24)):
            c = Case(seqs, 4, 2, hd, vd, 64, 90, 6, dtype, seed=8, padding=[3])
            want = c.run()
            for name in ("k_pool", "v_pool"):
                pool = getattr(c, name)
                moved = torch.empty(pool.numel() + 2, dtype=dtype, device=DEV)[2:].view(pool.shape)
                setattr(c, name, moved.copy_(pool))
            got = c.run()
            c.check(got)
            assert float((got.float() - want.float()).abs().max()) < 0.05
        c = Case(seqs, 4, 2, 64, 64, 64, 90, 6, BF16, seed=8)
        c.k_pool = torch.empty(c.k_pool.numel() + 2, dtype=BF16, device=DEV)[2:].view(c.k_pool.shape)
        with pytest.raises(K().KernelError):
            c.run()


def test_large_scores_and_a_first_key_that_takes_all_the_weight():
    """Scores of a few hundred: the running maximum moves by far more than an exponential's range, up and down the walk."""
    for spread in (30.0, 200.0):
        for hd in (64, 128):
            c = Case([(0, 200), (400, 150)], 4, 2, hd, hd, 64, 100, 4, BF16, seed=3, spread=spread)
            got = c.run().double().cpu().view(c.rows, 4, hd)
            assert bool(torch.isfinite(got).all())
            row = 0
            for (h, n), q, (k, v) in zip(c.seqs, c.q, c.kv):
                want = S.attention(q.double(), k.double(), v.double(), torch.arange(h, h + n), 100, 4, c.scale)[0]
                assert float((got[row:row + n] - want).abs().max()) < 2 ** -7 * float(want.abs().max()) + spread * 2e-4
                row += n


def test_first_positions_without_a_window_or_beyond_the_sequence_are_the_whole_of_it():
    for seqs in (DECODE, CHUNKS):
        for hd in (64, 128, 48):
            c = Case(seqs, 4, 2, hd, hd, 64, 0, 0, BF16, seed=2)
            whole = c.run()
            c.first = 77
            assert torch.equal(whole, c.run())          # no window: first has no effect
            c.window, c.first = 10, 5000
            c.check(c.run())
            assert float((c.run().float() - whole.float()).abs().max()) < 0.05


@pytest.mark.parametrize("seqs", [DECODE, CHUNKS])
@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 128), (BF16, 32), (F32, 48)])
def test_more_first_positions_than_32_bits_count(seqs, dtype, hd):
    c = Case(seqs, 4, 2, hd, hd, 64, 0, 0, dtype, seed=3)
    c.window = 10
    for c.first in (2 ** 31 - 1, 2 ** 31, 2 ** 33 + 5):
        c.check(c.run())


def test_offsets_beyond_32_bits():
    """Pools of more than 2^31 numbers, the sequences' pages at their end."""
    for hd, vd, seqs in ((64, 64, DECODE[:6]), (64, 64, CHUNKS[:4]), (128, 128, CHUNKS[:4]), (64, 32, CHUNKS[:4])):
        nkv = 8
        base = 2 ** 31 // (nkv * 64 * hd) + 1
        c = Case(seqs, 16, nkv, hd, vd, 64, 90, 5, BF16, base_page=base)
        c.check(c.run())
        del c
        torch.cuda.empty_cache()


@pytest.mark.parametrize("blocks", [0, 1, 2, 3, 8])
@pytest.mark.parametrize("dtype,nh,nkv,hd,vd,page", [(F32, 8, 2, 64, 64, 64), (F32, 3, 3, 128, 128, 32), (F32, 10, 2, 80, 48, 128), (F32, 4, 2, 33, 7, 64),
                                                     (F32, 2, 1, 256, 256, 64), (F32, 34, 1, 16, 40, 64), (BF16, 4, 2, 80, 80, 32), (BF16, 6, 2, 33, 50, 64)])
@pytest.mark.parametrize("window,first", [(1, 1), (64, 64), (300, 33), (33, 1000), (900, 4)])
def test_chunks_whose_rows_go_in_tiles(blocks, dtype, nh, nkv, hd, vd, page, window, first, monkeypatch):
    monkeypatch.setattr(K(), "STREAM_TILE_WORK", 0)
    c = Case(CHUNKS + [(5, 0), (700, 9)], nh, nkv, hd, vd, page, window, first, dtype, seed=5, padding=(2,))
    try:
        K().set_stream_attention_splits(blocks)
        c.check(c.run())
    finally:
        K().set_stream_attention_splits(0)


@pytest.mark.parametrize("dtype,hd,vd", [(F32, 64, 64), (F32, 48, 24), (BF16, 80, 72)])
def test_rows_in_tiles_with_slopes_sinks_and_gates(dtype, hd, vd, monkeypatch):
    """The same as rows one by one, up to roundings; an infinity that one row sees stays out of the rows that do not see it."""
    c = Case(CHUNKS, 6, 2, hd, vd, 32, 60, 9, dtype, seed=8)
    g = torch.Generator().manual_seed(3)
    slopes, sinks = torch.rand(6, generator=g).to(DEV), torch.randn(6, generator=g).to(DEV)
    for width in (6, 6 * vd):
        gate = torch.randn(c.rows, width, generator=g).to(dtype).to(DEV)
        one = c.run(slopes=slopes, sinks=sinks, gate=gate).float()
        with monkeypatch.context() as m:
            m.setattr(K(), "STREAM_TILE_WORK", 0)
            tiles = c.run(slopes=slopes, sinks=sinks, gate=gate).float()
        assert float((one - tiles).abs().max()) <= (2 ** -7 if dtype == BF16 else 2 ** -16) * float(one.abs().max())
    at = int(c.table[4, 530 // 32])      # a value that the rows up to 59 positions behind 530 see
    c.v_pool[at, :, :, 530 % 32] = float("inf")
    monkeypatch.setattr(K(), "STREAM_TILE_WORK", 0)
    out = c.run()
    row = sum(n for _, n in CHUNKS[:4])
    seen = torch.zeros(c.rows, dtype=torch.bool)
    seen[row + 530 - 517:row + 33] = True
    assert torch.isfinite(out.cpu().float()).all(1).eq(~seen).all()


@pytest.mark.parametrize("seqs", [DECODE, CHUNKS])
@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 128), (F32, 48)])
def test_rows_that_begin_anywhere(seqs, dtype, hd):
    """q and out one number behind a 16-byte boundary."""
    c = Case(seqs, 8, 2, hd, hd, 64, 100, 70, dtype, seed=21)
    q = torch.empty(1 + c.qd.numel(), dtype=dtype, device=DEV)[1:].view(c.qd.shape)
    q.copy_(c.qd)
    c.qd = q
    out = torch.full((1 + c.rows * 8 * hd,), float("nan"), dtype=dtype, device=DEV)[1:].view(c.rows, 8 * hd)
    K().attention(out, c.qd, c.k_pool, c.v_pool, c.table, c.batch, 8, 2, hd, 64, 100, c.scale, vd=hd, first=70)
    c.check(out)


def test_on_another_stream():
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c = Case(CHUNKS, 8, 2, 64, 64, 64, 100, 4, BF16)
        d = Case(DECODE, 8, 2, 64, 64, 64, 100, 4, BF16)
        a, b = c.run(), d.run()
    st.synchronize()
    c.check(a)
    d.check(b)


def test_attention_refuses():
    c = Case(DECODE, 4, 2, 64, 64, 64, 100, 4, BF16)
    c.first = -1
    with pytest.raises(K().KernelError):
        c.run(n_splits=1)


# ---- tables ----------------------------------------------------------------------------------------------------------
class Tables:
    def __init__(self, n_pages, n_slots, width, page, window, first):
        self.page, self.window, self.first, self.width = page, window, first, width
        self.lens, self.kept = words([0] * n_slots), words([-(-first // page)] * n_slots)
        self.pages = torch.full((n_slots, width), -1, dtype=torch.int32, device=DEV)
        self.free = words(list(range(n_pages - 1, -1, -1)))
        self.counts = words([n_pages, 77])

    def tables(self, slots, qlens, n_rows, width=None):
        B = len(slots)
        fill = lambda *s: torch.full(s, -123, dtype=torch.int32, device=DEV)
        o = {"table": fill(B, width or self.width), "slot_map": fill(n_rows), "row_seq": fill(n_rows), "row_pos": fill(n_rows),
             "slot": fill(B), "qlen": fill(B), "pos0": fill(B), "qstart": fill(B)}
        K().stream_tables(o["table"], o["slot_map"], o["row_seq"], o["row_pos"], o["slot"], o["qlen"], o["pos0"], o["qstart"], words(slots),
                          words(qlens), self.lens, self.pages, self.free, self.counts, self.page)
        return o

    def advance(self, o):
        K().stream_advance(o["slot"], o["qlen"], self.lens, self.kept, self.pages, self.free, self.counts, self.page, self.window, self.first)

    def release(self, slots):
        K().stream_release(words(slots), self.lens, self.kept, self.pages, self.free, self.counts, self.page, self.first)

    def same_as(self, plain):
        assert self.lens.tolist() == plain.lens
        assert torch.equal(self.pages.cpu(), torch.from_numpy(S.as_table(plain.lists, self.width)))
        n = int(self.counts[0])
        assert n == len(plain.free) and self.free[:n].tolist() == plain.free


def same_tables(o, t, slots, qlens):
    assert o["slot"].tolist() == list(slots) and o["qlen"].tolist() == list(qlens)
    for name in ("slot_map", "row_seq", "row_pos", "pos0", "qstart"):
        assert o[name].tolist() == t[name], name
    assert torch.equal(o["table"].cpu(), torch.from_numpy(S.as_table(t["table"], o["table"].shape[1])))


@pytest.mark.parametrize("n_slots,page,window,first,long", [
    (1, 64, 100, 4, 40), (5, 32, 1, 1, 90), (40, 64, 200, 65, 300), (300, 64, 0, 0, 70), (300, 128, 500, 200, 20), (1500, 32, 64, 0, 60),
    (1030, 64, 4096, 64, 9)])
def test_tables_over_many_steps(n_slots, page, window, first, long):
    """Steps of a random part of the slots, in random order, with padding and sequences without rows among them: decode steps, steps
    with prompts, steps that want more pages than there are; sequences end and their slots are used again."""
    rng = np.random.default_rng(n_slots + page)
    width = 40
    n_pages = n_slots * 9 + 3
    d, plain = Tables(n_pages, n_slots, width, page, window, first), S.PlainTables(n_pages, n_slots, width, page, window, first)
    refused = 0
    for step in range(24):
        some = rng.permutation(n_slots)[: max(1, int(rng.integers(1, n_slots + 1)))]
        slots = [int(s) if rng.random() < 0.9 else -1 for s in some]
        qlens = [int(rng.integers(0, long)) if step % 3 == 0 else 1 for _ in slots]
        want = plain.tables(slots, qlens, sum(qlens))
        o = d.tables(slots, qlens, sum(qlens))
        if isinstance(want, int):
            refused += 1
            assert int(d.counts[1]) == want
            assert o["slot"].tolist() == [-1] * len(slots) and o["qlen"].tolist() == [0] * len(slots)
            assert bool((o["slot_map"] == -1).all()) and bool((o["table"] == -1).all())
            if o["row_seq"].numel():
                assert int(o["row_seq"].min()) >= 0 and int(o["row_seq"].max()) < len(slots)
            d.advance(o)
            d.same_as(plain)
            gone = sorted({s for s in slots if s >= 0})
            d.release(gone + [-1])
            plain.release(gone)
        else:
            assert int(d.counts[1]) == 0
            same_tables(o, want, slots, qlens)
            again = d.tables(slots, qlens, sum(qlens))      # nothing but `advance` moves the state
            assert all(torch.equal(o[k], again[k]) for k in o)
            d.advance(o)
            plain.advance(slots, qlens, want)
        d.same_as(plain)
    d.release(list(range(n_slots)))
    plain.release(list(range(n_slots)))
    d.same_as(plain)
    assert int(d.counts[0]) == n_pages


def test_a_step_that_cannot_be_laid_out_changes_nothing():
    d, plain = Tables(6, 3, 4, 32, 0, 0), S.PlainTables(6, 3, 4, 32, 0, 0)
    o, t = d.tables([2, 0], [33, 40], 73), plain.tables([2, 0], [33, 40], 73)
    same_tables(o, t, [2, 0], [33, 40])
    d.advance(o)
    plain.advance([2, 0], [33, 40], t)
    for slots, qlens, rows, width, status in (([0, 1, 2], [1, 97, 1], 99, 4, 2), ([0], [89], 89, 4, -1), ([0], [30], 30, 2, -1),
                                              ([0, 1], [1, 1], 3, 4, -2), ([0, 3], [1, 1], 2, 4, -3), ([-2], [1], 1, 4, -3), ([0, 1], [2, -1], 1, 4, -3),
                                              ([1], [2 ** 31 - 1], 5, 4, -1)):
        assert plain.tables(slots, qlens, rows, width) == status
        o = d.tables(slots, qlens, rows, width)
        assert int(d.counts[1]) == status
        assert o["slot"].tolist() == [-1] * len(slots) and o["qlen"].tolist() == [0] * len(slots) and bool((o["slot_map"] == -1).all())
        d.advance(o)
        d.same_as(plain)
    d.release([-1, 7, -5])                              # no such slots
    d.same_as(plain)
    o, t = d.tables([0, 1], [1, 2], 3, width=3), plain.tables([0, 1], [1, 2], 3)
    same_tables(o, t, [0, 1], [1, 2])


def test_row_counts_whose_sum_goes_round():
    """Padding with row counts that add up to 2^32 more than the step's rows, and a sequence among them."""
    top = 2 ** 31 - 1
    for slots, qlens, rows in (([-1, -1, -1, 1], [top, top, 2, 7], 7), ([-1, 0, -1, -1], [top, 3, top, 2], 3), ([-1] * 600 + [2], [2 ** 23] * 512 + [0] * 88 + [4], 4)):
        d = Tables(6, 3, 4, 32, 0, 0)
        o = d.tables(slots, qlens, rows)
        assert int(d.counts[1]) == -2
        assert o["slot"].tolist() == [-1] * len(slots) and o["qlen"].tolist() == [0] * len(slots) and bool((o["slot_map"] == -1).all())
        d.advance(o)
        d.same_as(S.PlainTables(6, 3, 4, 32, 0, 0))


def test_tables_without_rows_and_without_sequences():
    d = Tables(6, 3, 4, 32, 0, 0)
    o = d.tables([0, -1], [0, 0], 0)
    assert o["slot"].tolist() == [0, -1] and o["qstart"].tolist() == [0, 0] and bool((o["table"] == -1).all()) and int(d.counts[1]) == 0
    d.advance(o)
    assert d.lens.tolist() == [0, 0, 0] and int(d.counts[0]) == 6
    o = d.tables([], [], 0)
    d.advance(o)


def test_tables_refuse():
    d = Tables(6, 3, 4, 32, 0, 0)
    k = K()
    i = lambda n: words([0] * n)
    good = dict(table=torch.zeros(2, 4, dtype=torch.int32, device=DEV), slot_map=i(5), row_seq=i(5), row_pos=i(5), step_slot=i(2), step_qlen=i(2),
                pos0=i(2), qstart=i(2), seq_slot=i(2), seq_qlen=i(2), lens=d.lens, pages=d.pages, free=d.free, counts=d.counts, page_size=32)
    for name, bad in (("row_pos", i(4)), ("qstart", i(3)), ("table", torch.zeros(3, 4, dtype=torch.int32, device=DEV)), ("lens", i(2)),
                      ("seq_slot", i(2).long()), ("counts", i(3)), ("pages", d.pages.t()), ("page_size", 0), ("slot_map", torch.zeros(5, dtype=torch.int32))):
        with pytest.raises(k.KernelError):
            k.stream_tables(**dict(good, **{name: bad}))
    with pytest.raises(k.KernelError):
        k.stream_advance(i(2), i(3), d.lens, d.kept, d.pages, d.free, d.counts, 32)
    with pytest.raises(k.KernelError):
        k.stream_advance(i(2), i(2), d.lens, d.kept, d.pages, d.free, d.counts, 32, window=-1)
    with pytest.raises(k.KernelError):
        k.stream_release(i(2), d.lens, i(1), d.pages, d.free, d.counts, 32)


# ---- stores ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nkv,hd,vd,page,shift", [(8, 64, 64, 64, 0), (2, 128, 128, 64, 0), (3, 80, 48, 32, 0), (1, 33, 7, 32, 1), (4, 64, 32, 128, 3), (1, 1, 1, 64, 0),
                                                  (2, 200, 256, 64, 0)])
@pytest.mark.parametrize("seqs", [[(0, 1)], [(5, 1), (64, 1), (127, 1), (31, 1)], [(0, 200), (63, 70), (10, 5)], [(7, 1000)]])
def test_stores_by_slot_map(dtype, nkv, hd, vd, page, shift, seqs):
    """Rows of a fused projection (also ones that begin in the middle of 16 bytes), some of them nowhere; everything else in the pools stays."""
    rng = np.random.default_rng(1)
    lists, n_pages = S.random_lists(rng, [h + n for h, n in seqs], page)
    slots = np.array([l[t // page] * page + t % page for (h, n), l in zip(seqs, lists) for t in range(h, h + n)], dtype=np.int32)
    M = len(slots)
    slots[rng.random(M) < 0.1] = -1
    g = torch.Generator().manual_seed(2)
    proj = torch.randn(M, shift + 5 + nkv * (hd + vd), generator=g).to(dtype).to(DEV)
    k, v = proj[:, shift:shift + nkv * hd], proj[:, shift + nkv * hd:shift + nkv * (hd + vd)]
    kp, vp = torch.randn(n_pages, nkv, page, hd, generator=g).to(dtype), torch.randn(n_pages, nkv, vd, page, generator=g).to(dtype)
    kd, vdev = kp.to(DEV), vp.to(DEV)
    K().store_rows(kd, vdev, k, v, words(slots))
    kc, vc = k.cpu().view(M, nkv, hd), v.cpu().view(M, nkv, vd)
    for m, s in enumerate(slots):
        if s >= 0:
            kp[s // page, :, s % page] = kc[m]
            vp[s // page, :, :, s % page] = vc[m]
    assert torch.equal(kd.cpu(), kp) and torch.equal(vdev.cpu(), vp)


@pytest.mark.parametrize("hd", [64, 40])
def test_stores_of_rows_in_any_order(hd):
    """A slot map whose rows are neither consecutive nor in order."""
    nkv, page, n_pages, M = 2, 64, 9, 300
    g = torch.Generator().manual_seed(2)
    slots = torch.randperm(n_pages * page, generator=g)[:M].to(torch.int32)
    k, v = (torch.randn(M, nkv * hd, generator=g).to(BF16) for _ in range(2))
    kd, vdev = torch.zeros(n_pages, nkv, page, hd, dtype=BF16, device=DEV), torch.zeros(n_pages, nkv, hd, page, dtype=BF16, device=DEV)
    K().store_rows(kd, vdev, k.to(DEV), v.to(DEV), slots.to(DEV))
    want_k, want_v = torch.zeros(kd.shape, dtype=BF16), torch.zeros(vdev.shape, dtype=BF16)
    s = slots.long()
    want_k[s // page, :, s % page] = k.view(M, nkv, hd)
    want_v[s // page, :, :, s % page] = v.view(M, nkv, hd)
    assert torch.equal(kd.cpu(), want_k) and torch.equal(vdev.cpu(), want_v)


def test_stores_beyond_32_bits_and_outside_the_pool():
    nkv, hd, page = 8, 64, 64
    n_pages = 2 ** 31 // (nkv * page * hd) + 2
    kd, vdev = (torch.zeros(n_pages, nkv, page, hd, dtype=BF16, device=DEV) for _ in range(2))
    k = torch.randn(3, nkv * hd).to(BF16).to(DEV)
    K().store_rows(kd, vdev, k, k, words([n_pages * page - 1, n_pages * page, 3]))      # the second lies outside: nowhere
    assert torch.equal(kd[-1, :, -1].reshape(-1), k[0]) and torch.equal(vdev.view(n_pages, nkv, hd, page)[-1, :, :, -1].reshape(-1), k[0])
    assert torch.equal(kd[0, :, 3].reshape(-1), k[2])
    assert int((kd != 0).sum()) == int((k[[0, 2]] != 0).sum())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [5, 500])
def test_stores_into_pools_that_begin_anywhere(dtype, M):
    """Pools one number behind a 16-byte boundary, rows whose places follow one another."""
    nkv, hd, page, n_pages = 2, 64, 64, 9
    at = lambda *shape: torch.zeros(1 + math.prod(shape), dtype=dtype, device=DEV)[1:].view(shape)
    kd, vdev = at(n_pages, nkv, page, hd), at(n_pages, nkv, hd, page)
    k, v = torch.randn(M, nkv * hd).to(dtype), torch.randn(M, nkv * hd).to(dtype)
    K().store_rows(kd, vdev, k.to(DEV), v.to(DEV), words(np.arange(2, 2 + M)))
    want_k, want_v = torch.zeros(kd.shape, dtype=dtype), torch.zeros(vdev.shape, dtype=dtype)
    s = torch.arange(2, 2 + M)
    want_k[s // page, :, s % page] = k.view(M, nkv, hd)
    want_v[s // page, :, :, s % page] = v.view(M, nkv, hd)
    assert torch.equal(kd.cpu(), want_k) and torch.equal(vdev.cpu(), want_v)


def test_stores_refuse():
    kd, vd_ = torch.zeros(4, 2, 32, 16, dtype=BF16, device=DEV), torch.zeros(4, 2, 8, 32, dtype=BF16, device=DEV)
    k, v, s = torch.zeros(3, 32, dtype=BF16, device=DEV), torch.zeros(3, 16, dtype=BF16, device=DEV), words([0, 1, 2])
    bad = [(kd, vd_, k.float(), v, s), (kd, vd_, k[:2], v, s), (kd, vd_, k, v[:, :8], s), (kd, vd_, k, v, s.long()), (kd, vd_.transpose(2, 3), k, v, s),
           (kd[:3], vd_, k, v, s), (kd, vd_, torch.zeros(3, 64, dtype=BF16, device=DEV)[:, ::2], v, s), (kd.half(), vd_.half(), k.half(), v.half(), s),
           (kd, vd_, k.cpu(), v, s)]
    for args in bad:
        with pytest.raises(K().KernelError):
            K().store_rows(*args)
    K().store_rows(kd, vd_, k[:0], v[:0], s[:0])


# ---- together ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,nh,nkv,hd,window,first", [(BF16, 8, 2, 64, 100, 4), (BF16, 4, 2, 128, 64, 70), (F32, 4, 2, 48, 33, 5)])
def test_a_decode_step_replayed_as_a_graph_goes_on_by_itself(dtype, nh, nkv, hd, window, first):
    """Prompts in one step, then one captured decode step replayed over several windows: the sequences advance, take and give back pages
    without the host, and every step's result is that of the whole history."""
    from lastengine_b200.cache import StreamCache
    B, steps = 3, 200
    pages_each = -(-first // 64) + -(-window // 64) + 1
    cache = StreamCache(2, nkv, hd, max_seqs=4, max_tokens=64 * (B * pages_each + 6), max_len=2048, window=window, first=first, dtype=dtype, device=DEV)
    slots = [cache.open() for _ in range(B)]
    g = torch.Generator().manual_seed(4)
    n0 = [70, 1, 130]
    total = [n + steps for n in n0]
    qs, ks, vs = ([torch.randn(t, w, generator=g).to(dtype) for t in total] for w in (nh * hd, nkv * hd, nkv * hd))
    prompt = cache.plan(B, sum(n0), max(n0))
    prompt.set(slots, n0)
    cache.begin(prompt)
    cat = lambda x: torch.cat([t[:n] for t, n in zip(x, n0)]).to(DEV)
    out = torch.empty(sum(n0), nh * hd, dtype=dtype, device=DEV)
    cache.store(1, prompt, cat(ks), cat(vs))
    cache.attend(1, prompt, out, cat(qs), nh)
    cache.check()

    def check(got, at):
        for b in range(B):
            n = at[b] + 1
            want, mass, size = S.attention(qs[b][at[b]:n].double().view(1, nh, hd), ks[b][:n].double().view(n, nkv, hd),
                                           vs[b][:n].double().view(n, nkv, hd), torch.tensor([at[b]]), window, first, hd ** -0.5)
            tol = (2 ** -8 * (1 + 2 ** -6) if dtype == BF16 else 2 ** -18) * (want.abs() + mass) + 2 * mass * hd * 2 ** -22 * size
            assert bool(((got[b].double().cpu().view(1, nh, hd) - want).abs() <= tol).all()), (at, b)

    ends = np.cumsum(n0) - 1
    check(out[ends.tolist()], [n - 1 for n in n0])
    step = cache.plan(B, B, 1)
    step.set(slots, [1] * B)
    q, k, v, o = (torch.zeros(B, w, dtype=dtype, device=DEV) for w in (nh * hd, nkv * hd, nkv * hd, nh * hd))

    def one():
        cache.begin(step)
        cache.store(1, step, k, v)
        cache.attend(1, step, o, q, nh)

    saved = cache.state.clone()
    one()                                               # warm: then taken back
    cache.state.copy_(saved)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one()
    for i in range(steps):
        for dst, src in ((q, qs), (k, ks), (v, vs)):
            dst.copy_(torch.stack([src[b][n0[b] + i] for b in range(B)]))
        graph.replay()
        if i % 9 == 0 or i == steps - 1:
            check(o, [n + i for n in n0])
    cache.check()
    assert cache.lengths(slots) == total
    held = sum(int((cache.pages[s] >= 0).sum()) for s in slots)
    assert held <= B * pages_each and int(cache.counts[0]) + held == cache.free.numel()
    cache.close(slots[:2])
    cache.close(slots[2:])
    assert sorted(cache.free.tolist()) == list(range(cache.free.numel())) and bool((cache.pages == -1).all())


def test_a_step_without_room_is_reported_and_touches_no_cache():
    from lastengine_b200.cache import CacheError, CacheFull, StreamCache
    cache = StreamCache(1, 2, 64, max_seqs=2, max_tokens=192, max_len=256, device=DEV)
    a, b = cache.open(), cache.open()
    rows = lambda n: torch.randn(n, 128, device=DEV).to(BF16)
    for counts, error in ([([64, 64], None), ([1, 1], CacheFull), ([200, 1], CacheError), ([1, 0], None)]):
        step = cache.plan(2, sum(counts), max(counts))
        step.set([a, b], counts)
        cache.begin(step)
        before = cache.k.clone()
        cache.store(0, step, rows(sum(counts)), rows(sum(counts)))
        out = torch.zeros(sum(counts), 256, dtype=BF16, device=DEV)
        cache.attend(0, step, out, torch.randn(sum(counts), 256, device=DEV).to(BF16), 4)
        if error is None:
            cache.check()
            assert bool(torch.isfinite(out).all()) and not torch.equal(before, cache.k)
        else:
            with pytest.raises(error):
                cache.check()
            assert torch.equal(before, cache.k)
    assert cache.lengths([a, b]) == [65, 64]


C5 = dict(TINY_C, sliding_window=24, sliding_window_first=5)
D9 = dict(TINY_D, sliding_window=20, sliding_window_first=9)


@pytest.mark.parametrize("name,cfg", [("C", C5), ("D", D9)])
@pytest.mark.parametrize("dtype,bf16,tol", [("float32", False, H.TOL_F32), ("bfloat16", True, H.TOL_BF16)])
def test_a_model_whose_windowed_layers_see_first_positions(name, cfg, dtype, bf16, tol, tmp_path, monkeypatch):
    from lastengine_b200 import Engine, SamplingParams
    d = H.make_model_dir(cfg, 3, str(tmp_path), freq_factors=name == "D")
    eng = Engine.from_pretrained(d, dtype=dtype, max_tokens=2048)
    requests = H.requests_for(cfg, [5, 40, 150, 201], 7)
    orig = P.attention
    # layers without a window are as they were
    part = S.lfm3_attention(cfg["sliding_window_first"])
    monkeypatch.setattr(P, "attention", lambda *a, **k: part(*a, **k) if k.get("window") else orig(*a, **k))
    for r in requests:
        want, margins = H.plain_logits_and_margins(cfg, d, r, bf16)
        keep = H.decided(margins, bf16)
        for got in (H.run_whole(eng, r), H.run_tail(eng, r)):
            assert H.rel_err(got[keep], want[keep]) <= tol
    # a sequence goes on from its bytes as it would have
    s = eng.new_sequence()
    eng.step([s], [requests[3][:180]])
    saved = eng.export_sequence(s)
    t = eng.import_sequence(saved)
    a, b = (eng.step([x], [requests[3][180:]], [list(range(21))]).float().cpu().clone() for x in (s, t))
    assert torch.equal(a, b)
    eng.release(s)
    eng.release(t)
    params = SamplingParams(temperature=0.0)
    with_graphs = eng.generate(requests, params, max_new_tokens=40, use_graphs=True).tokens
    assert with_graphs == eng.generate(requests, params, max_new_tokens=40, use_graphs=False).tokens


def test_the_example_runs():
    import os
    import subprocess
    import sys
    env = dict(os.environ, PYTHONPATH=H.ROOT)
    r = subprocess.run([sys.executable, os.path.join(H.ROOT, "examples", "endless_stream.py"), "--streams", "3", "--steps", "500", "--window", "130",
                        "--prompt", "70", "--layers", "2"], env=env, cwd=H.ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    held = [int(x) for x in r.stdout.split("[")[1].split("]")[0].split(",")]
    assert max(held[2:]) <= 3 * 5 and "571 positions" in r.stdout
