"""Steps with first positions at the edges of what single kernels take: very many rows, rows and pools that begin anywhere."""
import types

import pytest
import torch

import harness as H  # noqa: F401  (path setup)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def K():
    from lastengine_b200.ops import kernels
    return kernels


def at(t, behind):
    """t, `behind` numbers behind a 16-byte boundary."""
    return torch.empty(behind + t.numel(), dtype=t.dtype, device=DEV)[behind:].view(t.shape).copy_(t)


def one_sequence(M, nh, hd, vd, page, dtype, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)
    n = -(-M // page)
    word = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    batch = types.SimpleNamespace(n_rows=M, n_seqs=1, max_qlen=M, max_kvlen=M, row_seq=torch.zeros(M, dtype=torch.int32, device=DEV),
                                  row_pos=torch.arange(M, dtype=torch.int32, device=DEV), seq_slot=word([0]), seq_pos0=word([0]), seq_qstart=word([0]),
                                  seq_qlen=word([M]))
    return batch, rand(M, nh * hd), rand(n, 1, page, hd), rand(n, 1, vd, page), torch.arange(n, dtype=torch.int32, device=DEV)[None]


@pytest.mark.parametrize("dtype,nh,hd,vd,page,rows_at,pools_at", [(BF16, 1, 32, 32, 32, 1, 0), (BF16, 1, 32, 32, 32, 0, 0), (BF16, 1, 64, 64, 64, 4, 0), (F32, 1, 32, 16, 32, 1, 0),
                                                                  (F32, 1, 32, 16, 32, 0, 1), (BF16, 66, 8, 8, 32, 1, 0)])
def test_more_rows_than_a_grid_s_second_dimension(dtype, nh, hd, vd, page, rows_at, pools_at):
    M, window, first = 70001, 30, 5
    batch, q, k, v, table = one_sequence(M, nh, hd, vd, page, dtype)
    qd, kd, vd_ = at(q, rows_at), at(k, pools_at), at(v, pools_at)
    out = at(torch.full((M, nh * vd), float("nan"), dtype=dtype, device=DEV), rows_at)
    K().attention(out, qd, kd, vd_, table, batch, nh, 1, hd, page, window, hd ** -0.5, vd=vd, first=first)
    K().check_device_status()
    kk, vv = k[:, 0].reshape(-1, hd)[:M].double(), v[:, 0].transpose(1, 2).reshape(-1, vd)[:M].double()
    p = torch.arange(M, device=DEV)
    # the window's positions, then the first ones that lie before it
    back = p[:, None] - torch.arange(window, device=DEV)
    t = torch.cat([back, torch.arange(first, device=DEV).expand(M, first)], 1)
    ok = torch.cat([back >= 0, torch.arange(first, device=DEV)[None] <= p[:, None] - window], 1)
    t = t.clamp(min=0)
    for h in range(0, nh, 13):
        qq = q[:, h * hd:(h + 1) * hd].double()
        s = torch.einsum("md,mtd->mt", qq, kk[t]) * hd ** -0.5
        size = torch.einsum("md,mtd->mt", qq.abs(), kk[t].abs()).amax(1, keepdim=True) * hd ** -0.5
        w = torch.softmax(s.masked_fill(~ok, float("-inf")), -1)
        want, mass = torch.einsum("mt,mtd->md", w, vv[t]), torch.einsum("mt,mtd->md", w, vv[t].abs())
        # the roundings of tests/test_gpu_stream.py
        if dtype == BF16:
            bound = 2 ** -8 * (1 + 2 ** -6) * (want.abs() + mass) + 2 * mass * (hd * 2 ** -22 * size + 35 * 2 ** -24 + 2 ** -18)
        else:
            bound = want.abs() * 2 ** -22 + 2 * mass * ((hd + 8) * 2 ** -24 * size + 35 * 2 ** -24 + 2 ** -20)
        assert bool(((out[:, h * vd:(h + 1) * vd].double() - want).abs() <= bound + 1e-30).all()), h


@pytest.mark.parametrize("M,B", [(4, 4), (6, 2), (40, 2), (300, 1)])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_addresses_that_the_kernels_for_all_rows_do_not_take_are_refused(M, B, hd):
    """Without first positions: nothing is launched on rows or pools off the boundaries that 16-byte loads want."""
    word = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    n = M // B
    batch = types.SimpleNamespace(n_rows=M, n_seqs=B, max_qlen=n, max_kvlen=n, row_seq=word([i // n for i in range(M)]), row_pos=word([i % n for i in range(M)]),
                                  seq_slot=word(list(range(B))), seq_pos0=word([0] * B), seq_qstart=word([b * n for b in range(B)]), seq_qlen=word([n] * B))
    pages = -(-n // 64)
    table = torch.arange(B * pages, dtype=torch.int32, device=DEV).view(B, pages)
    q, k, v = (torch.randn(s, device=DEV).to(BF16) for s in ((M, 2 * hd), (B * pages, 1, 64, hd), (B * pages, 1, hd, 64)))
    run = lambda q, k, v: K().attention(torch.empty(M, 2 * hd, dtype=BF16, device=DEV), q, k, v, table, batch, 2, 1, hd, 64, 0, hd ** -0.5)
    run(q, k, v)
    for args in ((at(q, 1), k, v), (q, at(k, 4), v), (q, k, at(v, 1))):
        with pytest.raises(K().KernelError):
            run(*args)
    torch.cuda.synchronize()


@pytest.mark.parametrize("new", [1, 5, 150])
@pytest.mark.parametrize("dtype,nh,nkv,hd,page", [(BF16, 8, 2, 64, 64), (BF16, 3, 3, 128, 64), (BF16, 4, 2, 32, 32), (BF16, 2, 1, 72, 64), (F32, 4, 2, 48, 32)])
@pytest.mark.parametrize("first", [0, 70])
@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-30, 1e-22])
def test_scales_that_are_not_positive_or_next_to_nothing(new, dtype, nh, nkv, hd, page, first, scale):
    """What a row does not see has no weight, whatever the scores that it sees are multiplied by."""
    held, window, G = 250, 90, nh // nkv
    T = held + new
    word = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    rand = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)
    n = -(-T // page)
    q, k, v = rand(new, nh * hd), rand(n, nkv, page, hd), rand(n, nkv, hd, page)
    batch = types.SimpleNamespace(n_rows=new, n_seqs=1, max_qlen=new, max_kvlen=T, row_seq=word([0] * new), row_pos=word(list(range(held, T))),
                                  seq_slot=word([0]), seq_pos0=word([held]), seq_qstart=word([0]), seq_qlen=word([new]))
    out = torch.full((new, nh * hd), float("nan"), dtype=dtype, device=DEV)
    K().attention(out, q, k, v, torch.arange(n, dtype=torch.int32, device=DEV)[None], batch, nh, nkv, hd, page, window, scale, first=first)
    K().check_device_status()
    p, t = torch.arange(held, T, device=DEV)[:, None], torch.arange(T, device=DEV)[None]
    ok = (t <= p) & ((t > p - window) | (t < first))
    for h in range(nh):
        qq = q[:, h * hd:(h + 1) * hd].double()
        kk, vv = k[:, h // G].reshape(-1, hd)[:T].double(), v[:, h // G].transpose(1, 2).reshape(-1, hd)[:T].double()
        w = torch.softmax((qq @ kk.T * scale).masked_fill(~ok, float("-inf")), -1)
        size = (qq.abs() @ kk.abs().T * abs(scale)).amax(1, keepdim=True)
        want, mass = w @ vv, w @ vv.abs()
        # the roundings of tests/test_gpu_stream.py
        if dtype == BF16:
            bound = 2 ** -8 * (1 + 2 ** -6) * (want.abs() + mass) + 2 * mass * (hd * 2 ** -22 * size + T * 2 ** -24 + 2 ** -18)
        else:
            bound = want.abs() * 2 ** -22 + 2 * mass * ((hd + 8) * 2 ** -24 * size + T * 2 ** -24 + 2 ** -20)
        assert bool(((out[:, h * hd:(h + 1) * hd].double() - want).abs() <= bound + 1e-30).all()), h
