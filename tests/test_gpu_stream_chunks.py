"""First positions beside chunks of positions (and beside a window within a chunk), and decode steps that norm, rotate and store their own
keys with first positions: every kernel, against plain arithmetic in double precision."""
import math
import types

import numpy as np
import pytest
import torch

import harness as H
import plain_lfm3 as P
import plain_stream as S
from tiny_configs import TINY_C

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def K():
    from lastengine_b200.ops import kernels
    return kernels


def words(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)


def start_of(p, window, chunk):
    """The first position that the row at p reads, its first positions aside."""
    return max(p + 1 - window if window > 0 else 0, p // chunk * chunk if chunk > 0 else 0, 0)


def sees(pos, t, window, chunk, first):
    lo = torch.tensor([start_of(int(p), window, chunk) for p in pos])
    return (t[None] <= pos[:, None]) & ((t[None] >= lo[:, None]) | (t[None] < first))


class Step:
    """Sequences of (positions held, rows brought): only positions that a row of the step sees are filled, everything else holds NaN, and
    pages that no row from the step's first on reads are given back (-1)."""

    def __init__(self, seqs, nh, nkv, hd, vd, page, window, chunk, first, dtype, seed=0, padding=()):
        rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.__dict__.update(seqs=seqs, nh=nh, nkv=nkv, hd=hd, vd=vd, page=page, window=window, chunk=chunk, first=first, dtype=dtype,
                             padding=set(padding), scale=hd ** -0.5)
        lists, n_pages = S.random_lists(rng, [h + n for h, n in seqs], page)
        self.k_pool = torch.full((n_pages, nkv, page, hd), float("nan"), dtype=dtype, device=DEV)
        self.v_pool = torch.full((n_pages, nkv, vd, page), float("nan"), dtype=dtype, device=DEV)
        self.q, self.kv = [], []
        for b, ((h, n), l) in enumerate(zip(seqs, lists)):
            q = torch.randn(n, nh, hd, generator=g).to(dtype)
            k, v = torch.randn(h + n, nkv, hd, generator=g).to(dtype), torch.randn(h + n, nkv, vd, generator=g).to(dtype)
            self.q.append(q)
            self.kv.append((k, v))
            if b in self.padding:
                continue
            seen = sees(torch.arange(h, h + n), torch.arange(h + n), window, chunk, first).any(0)
            for j, p in enumerate(l):
                at = torch.tensor([t for t in range(j * page, min((j + 1) * page, h + n)) if n and seen[t]], dtype=torch.long)
                if at.numel():
                    self.k_pool[p, :, at % page] = k[at].permute(1, 0, 2).to(DEV)
                    self.v_pool[p, :, :, at % page] = v[at].permute(1, 2, 0).to(DEV)
            for j in range(-(-first // page), min(len(l), start_of(h, window, chunk) // page)):
                l[j] = -1
        pos0, qlen = [0 if b in self.padding else h for b, (h, n) in enumerate(seqs)], [n for h, n in seqs]
        self.rows = sum(qlen)
        self.table = torch.from_numpy(S.as_table(lists, max(len(l) for l in lists))).to(DEV)
        self.batch = types.SimpleNamespace(
            n_rows=self.rows, n_seqs=len(seqs), max_qlen=max(qlen), max_kvlen=max(h + n for h, n in seqs),
            row_seq=words(np.repeat(np.arange(len(seqs)), qlen)), row_pos=words(np.concatenate([p + np.arange(n) for p, n in zip(pos0, qlen)])),
            seq_slot=words([-1 if b in self.padding else b for b in range(len(seqs))]), seq_pos0=words(pos0),
            seq_qstart=words(np.cumsum([0] + qlen[:-1])), seq_qlen=words(qlen))
        self.qd = torch.cat(self.q).reshape(self.rows, nh * hd).to(DEV)

    def run(self, n_splits=1, **kw):
        out = torch.full((self.rows, self.nh * self.vd), float("nan"), dtype=self.dtype, device=DEV)
        scratch = torch.full((self.rows * self.nh * n_splits * (max(self.hd, self.vd) + 2),), float("nan"), device=DEV) if n_splits > 1 else None
        K().attention(out, self.qd, self.k_pool, self.v_pool, self.table, self.batch, self.nh, self.nkv, self.hd, self.page, self.window,
                      self.scale, n_splits=n_splits, scratch=scratch, vd=self.vd, chunk=self.chunk, first=self.first, **kw)
        return out

    def check(self, out, slopes=None, sinks=None):
        """Roundings, each at its worst: bfloat16 weights and results 2^-8 of what they are; a score's sum over the head 2^-22 (float32: 2^-24) of
        its terms' magnitudes a term, which moves a weight by as much; sums over positions 2^-24 a term; exponentials 2^-20 (2^-18)."""
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
            t = torch.arange(h + n)
            ok = sees(torch.arange(h, h + n), t, self.window, self.chunk, self.first)
            for x in range(self.nh):
                k, v = (y[:, x // (self.nh // self.nkv)].double() for y in self.kv[b])
                q = self.q[b][:, x].double()
                s, size = q @ k.T * self.scale, (q.abs() @ k.abs().T * self.scale).masked_fill(~ok, 0.0).amax(-1, keepdim=True)
                if slopes is not None:
                    s = s - slopes[x] * (torch.arange(h, h + n)[:, None] - t)
                    size = size + slopes.abs().max() * (h + n) * 2 ** -4
                s = s.masked_fill(~ok, -math.inf)
                w = torch.softmax(s if sinks is None else torch.cat([s, torch.full((n, 1), float(sinks[x]), dtype=torch.float64)], 1), -1)[:, :h + n]
                want, mass = w @ v, w @ v.abs()
                T = min(h + n, (self.window or self.chunk) + self.first)
                if self.dtype == BF16:
                    bound = 2 ** -8 * (1 + 2 ** -6) * (want.abs() + mass) + 2 * mass * (self.hd * 2 ** -22 * size + T * 2 ** -24 + 2 ** -18)
                else:
                    bound = want.abs() * 2 ** -22 + 2 * mass * ((self.hd + 8) * 2 ** -24 * size + T * 2 ** -24 + 2 ** -20)
                off = (got[:, x] - want).abs()
                assert bool((off <= bound + 1e-30).all()), (b, h, n, x, float((off / (bound + 1e-30)).nan_to_num(1e9).max()))


SHAPES = [(0, 1, 1), (0, 33, 5), (0, 64, 64), (0, 64, 70), (0, 100, 4), (0, 100, 130), (0, 256, 33), (0, 48, 1000), (40, 100, 6), (100, 64, 9), (200, 256, 65)]
DECODE = [(0, 1), (31, 1), (32, 1), (63, 1), (64, 1), (99, 1), (100, 1), (127, 1), (200, 1), (511, 1), (512, 1), (700, 1), (1023, 1)]
CHUNKS = [(0, 1), (0, 70), (63, 2), (200, 130), (517, 33), (64, 64), (99, 2), (255, 3), (3, 300)]


@pytest.mark.parametrize("dtype,nh,nkv,hd,vd,page", [
    (BF16, 8, 2, 64, 64, 64), (BF16, 16, 1, 128, 128, 64), (BF16, 3, 1, 32, 32, 32), (BF16, 6, 6, 96, 96, 128), (BF16, 4, 2, 80, 80, 64),
    (BF16, 6, 2, 33, 65, 64), (BF16, 34, 2, 64, 64, 64), (F32, 4, 2, 64, 64, 64), (F32, 6, 2, 80, 48, 32), (F32, 5, 1, 256, 200, 64)])
@pytest.mark.parametrize("window,chunk,first", SHAPES)
def test_single_tokens(dtype, nh, nkv, hd, vd, page, window, chunk, first):
    c = Step(DECODE, nh, nkv, hd, vd, page, window, chunk, first, dtype, seed=window + chunk + first, padding=[4])
    c.check(c.run())
    c.check(c.run(n_splits=3))
    try:
        for n in (1, 2, 5, 8):
            K().set_stream_attention_splits(n)
            c.check(c.run())
    finally:
        K().set_stream_attention_splits(0)


@pytest.mark.parametrize("dtype,nh,nkv,hd,vd,page", [
    (BF16, 8, 2, 64, 64, 64), (BF16, 3, 3, 64, 64, 64), (BF16, 8, 2, 128, 128, 64), (BF16, 5, 1, 128, 128, 128), (BF16, 3, 1, 72, 40, 64),
    (BF16, 4, 2, 32, 32, 32), (BF16, 2, 2, 96, 96, 32), (BF16, 34, 2, 64, 64, 64), (BF16, 2, 1, 192, 192, 64), (F32, 4, 2, 64, 64, 64), (F32, 6, 2, 80, 48, 32)])
@pytest.mark.parametrize("window,chunk,first", SHAPES)
def test_chunks_of_tokens(dtype, nh, nkv, hd, vd, page, window, chunk, first, monkeypatch):
    c = Step(CHUNKS, nh, nkv, hd, vd, page, window, chunk, first, dtype, seed=window + chunk + first, padding=[5])
    c.check(c.run())
    try:
        for n in (1, 3, 8):      # blocks that share a tile's keys
            K().set_stream_attention_splits(n)
            c.check(c.run())
            with monkeypatch.context() as m:
                m.setattr(K(), "STREAM_TILE_WORK", 0)
                c.check(c.run())
    finally:
        K().set_stream_attention_splits(0)
    if vd == hd:
        c.check(c.run(wide=True))


@pytest.mark.parametrize("seqs", [DECODE, CHUNKS])
@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 32), (F32, 48)])
def test_slopes_and_sinks(seqs, dtype, hd):
    c = Step(seqs, 4, 2, hd, hd, 64, 0, 70, 40, dtype, seed=9)
    slopes, sinks = 2.0 ** -torch.arange(1, 5).float(), torch.randn(4, generator=torch.Generator().manual_seed(1))
    c.check(c.run(slopes=slopes.to(DEV), sinks=sinks.to(DEV)), slopes.double(), sinks.double())


@pytest.mark.parametrize("seqs", [DECODE, CHUNKS])
@pytest.mark.parametrize("window,chunk,first", SHAPES)
@pytest.mark.parametrize("dtype,hd,vd", [(F32, 48, 48), (BF16, 72, 24)])
def test_pools_that_begin_anywhere(seqs, window, chunk, first, dtype, hd, vd):
    """(the general kernel)"""
    c = Step(seqs, 4, 2, hd, vd, 64, window, chunk, first, dtype, seed=8, padding=[3])
    for name in ("k_pool", "v_pool"):
        pool = getattr(c, name)
        setattr(c, name, torch.empty(pool.numel() + 2, dtype=dtype, device=DEV)[2:].view(pool.shape).copy_(pool))
    c.check(c.run())


# ---- steps that norm, rotate and store their own keys ------------------------------------------------------------------
@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 64), (6, 2, 128), (5, 5, 64), (16, 1, 64)])
@pytest.mark.parametrize("window,chunk,first,gated", [(40, 0, 5, False), (100, 0, 64, True), (64, 0, 70, False), (0, 64, 3, True), (0, 100, 130, False), (50, 64, 9, False)])
def test_decode_steps_that_store_their_own_keys(nh, nkv, hd, window, chunk, first, gated):
    """The same bits as with the rotary kernel first, and the same cache, for any number of blocks or splits, a new position that is the first of
    all, the first or last place of a page or the first of a chunk; what lies outside a row's sight is NaN; against double precision."""
    page, theta, eps, scale = 64, 5e4, 1e-5, hd ** -0.5
    lens = [130, 1, 64, 65, 257, 7, 1025, 701]                 # after the step: the new token sits at len - 1
    slots = [0, 1, -1, 2, 3, 4, 5, 6]
    B, g = len(lens), torch.Generator().manual_seed(5)
    lists, n_pages = S.random_lists(np.random.default_rng(6), lens, page)
    kp0 = torch.full((n_pages, nkv, page, hd), float("nan"), dtype=BF16)
    vp0 = torch.full((n_pages, nkv, hd, page), float("nan"), dtype=BF16)
    for n, s, l in zip(lens, slots, lists):
        seen = sees(torch.tensor([n - 1]), torch.arange(n), window, chunk, first)[0]
        for t in range(n - 1):
            if s >= 0 and seen[t]:
                kp0[l[t // page], :, t % page] = torch.randn(nkv, hd, generator=g).to(BF16)
                vp0[l[t // page], :, :, t % page] = torch.randn(nkv, hd, generator=g).to(BF16)
    kp0, vp0 = kp0.to(DEV), vp0.to(DEV)
    table = torch.from_numpy(S.as_table([[-1 if -(-first // page) <= j < start_of(n - 1, window, chunk) // page else p for j, p in enumerate(l)]
                                         for n, l in zip(lens, lists)], max(map(len, lists)))).to(DEV)
    batch = types.SimpleNamespace(
        n_rows=B, n_seqs=B, max_qlen=1, max_kvlen=max(lens), row_seq=words(range(B)), row_pos=words([n - 1 if s >= 0 else 0 for n, s in zip(lens, slots)]),
        seq_slot=words(slots), seq_pos0=words([n - 1 if s >= 0 else 0 for n, s in zip(lens, slots)]), seq_qstart=words(range(B)), seq_qlen=words([1] * B))
    qkv = torch.randn(B, (nh + 2 * nkv) * hd + nh, generator=g).to(BF16).to(DEV)
    q_in, k_in = qkv[:, :nh * hd], qkv[:, nh * hd:(nh + nkv) * hd]
    v_in, gate = qkv[:, (nh + nkv) * hd:(nh + 2 * nkv) * hd], (qkv[:, (nh + 2 * nkv) * hd:] if gated else None)
    qn, kn = ((1 + 0.1 * torch.randn(hd, generator=g)).to(DEV) for _ in range(2))
    inv = torch.pow(torch.tensor(theta, dtype=torch.float64), -2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd).float().to(DEV)
    assert K().decode_attention_takes_raw(BF16, batch, B, nh, nkv, hd, page, inv, hd, True)

    def both(splits):
        scratch = torch.empty(B * nh * splits * (hd + 2), device=DEV) if splits > 1 else None
        kw = dict(gate=gate, n_splits=splits, scratch=scratch, chunk=chunk, first=first)
        kp_a, vp_a, kp_b, vp_b = kp0.clone(), vp0.clone(), kp0.clone(), vp0.clone()
        q_rot, want = (torch.empty(B, nh * hd, device=DEV, dtype=BF16) for _ in range(2))
        K().qk_rope_store(q_rot, q_in, k_in, v_in, kp_a, vp_a, table, batch, qn, kn, eps, inv, hd, True, nh, nkv, hd, page)
        K().attention(want, q_rot, kp_a, vp_a, table, batch, nh, nkv, hd, page, window, scale, **kw)
        got = torch.full_like(want, float("nan"))
        K().attention(got, None, kp_b, vp_b, table, batch, nh, nkv, hd, page, window, scale,
                      raw=K().RawQKV(q_in, k_in, v_in, qn, kn, eps, inv, hd, True), **kw)
        same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))
        assert same(kp_a, kp_b) and same(vp_a, vp_b) and not same(kp_a, kp0) and not same(vp_a, vp0)
        assert torch.equal(got, want), (splits, float((got.float() - want.float()).abs().max()))
        return got, kp_b, vp_b

    made = [both(1), both(2), both(5)]
    try:
        for n in (1, 2, 3, 8):
            K().set_stream_attention_splits(n)
            made.append(both(1))
    finally:
        K().set_stream_attention_splits(0)
    for got, kp, vp in made:
        got, kp, vp = got.double().cpu(), kp.double().cpu(), vp.double().cpu()
        for b, (n, s, l) in enumerate(zip(lens, slots, lists)):
            if s < 0:
                assert float(got[b].abs().max()) == 0.0
                continue
            at = [int(t) for t in torch.nonzero(sees(torch.tensor([n - 1]), torch.arange(n), window, chunk, first)[0])]
            k = torch.stack([kp[l[t // page], :, t % page] for t in at])
            v = torch.stack([vp[l[t // page], :, :, t % page] for t in at])
            row = qkv[b].double().cpu()
            turn = lambda x, w: P.rope(P.rms_norm(x, w.double().cpu(), eps), torch.tensor([n - 1]), hd, theta)[0]
            new = turn(row[nh * hd:(nh + nkv) * hd].view(1, nkv, hd), kn)
            # the rotation's angle is a float product of up to 1,025 radians: 2^-13 at the most, beside the rounding to bfloat16
            assert bool(((k[-1] - new).abs() <= 2 ** -8 * new.abs() + 2 ** -12 * new.abs().max()).all())
            assert torch.equal(v[-1], row[(nh + nkv) * hd:(nh + 2 * nkv) * hd].view(nkv, hd))
            q = P.round_bf16(turn(row[:nh * hd].view(1, nh, hd), qn))
            for h in range(nh):
                kk, vv = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
                size = float((kk.abs() @ q[h].abs()).max()) * scale
                w = torch.softmax(kk @ q[h] * scale, 0)
                o, mass = w @ vv, w @ vv.abs()
                if gated:
                    f = torch.sigmoid(row[(nh + 2 * nkv) * hd + h])
                    o, mass = o * f, mass * f
                # as elsewhere, and queries that the angle or another rounding moves by 2^-8
                bound = 2 ** -8 * (1 + 2 ** -6) * (o.abs() + mass) + 2 * mass * (2 ** -8 + hd * 2 ** -22) * size + 2 ** -16
                assert bool(((got[b].view(nh, hd)[h] - o).abs() <= bound).all()), (b, h)


REAL_HEADS = dict(TINY_C, num_attention_heads=32, num_key_value_heads=8, head_dim=64, rope_dim=64, sliding_window=24, sliding_window_first=5)
WIDE_HEADS = dict(TINY_C, num_attention_heads=6, num_key_value_heads=2, head_dim=128, rope_dim=128, sliding_window=70, sliding_window_first=9)


@pytest.mark.parametrize("name,cfg", [("32 heads of 64", REAL_HEADS), ("heads of 128", WIDE_HEADS)])
@pytest.mark.parametrize("dtype,bf16,tol", [("float32", False, H.TOL_F32), ("bfloat16", True, H.TOL_BF16)])
def test_a_model_whose_decode_steps_store_their_own_keys(name, cfg, dtype, bf16, tol, tmp_path, monkeypatch):
    """Heads and rotation of the sizes whose decode step is one launch from the projection to the heads' results."""
    from lastengine_b200 import Engine, SamplingParams
    d = H.make_model_dir(cfg, 3, str(tmp_path))
    eng = Engine.from_pretrained(d, dtype=dtype, max_tokens=2048)
    requests = H.requests_for(cfg, [5, 40, 150, 201], 7)
    orig, part = P.attention, S.lfm3_attention(cfg["sliding_window_first"])
    monkeypatch.setattr(P, "attention", lambda *a, **k: part(*a, **k) if k.get("window") else orig(*a, **k))
    raws, decode_raw = [], K()._attention_decode_raw
    monkeypatch.setattr(K(), "_attention_decode_raw", lambda *a, **k: (raws.append(a[-1]), decode_raw(*a, **k))[1])
    for r in requests:
        want, margins = H.plain_logits_and_margins(cfg, d, r, bf16)
        keep = H.decided(margins, bf16)
        for got in (H.run_whole(eng, r), H.run_tail(eng, r)):
            assert H.rel_err(got[keep], want[keep]) <= tol
    assert (cfg["sliding_window_first"] in raws) == bf16
    params = SamplingParams(temperature=0.0)
    with_graphs = eng.generate(requests, params, max_new_tokens=40, use_graphs=True).tokens
    assert with_graphs == eng.generate(requests, params, max_new_tokens=40, use_graphs=False).tokens
