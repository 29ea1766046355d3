"""A number that is not one stays so through every activation: in the epilogues of the products, whichever kernel takes them, and in the
activations' own kernels.  A row whose scale says that it could not be held in 8 bits must not come out of an activation as
plausible numbers."""
import pytest
import torch

import harness as H  # noqa: F401  (path setup)
import plain_e4m3 as P
from test_gpu_e4m3 import act_bound, gen, powers, whole_numbers

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
NAN = float("nan")


def K():
    from lastengine_b200.ops import kernels
    return kernels


def gates():
    k = K()
    return {"silu": k.gated_epilogue(k.SILU), "gelu_tanh": k.gated_epilogue(k.GELU_TANH), "clamped": k.gated_epilogue(k.CLAMPED_SIGMOID, 7.0, 1.702)}


# rows, columns, K, how far rows lie apart, and the form that takes them on 148 SMs (0: pairs; else rows of a tile | slices of K << 16)
PRODUCTS = {
    "a cluster a tile": (40, 160, 4096, 4096, 16 | 8 << 16), "tiles in a row": (20, 4128, 256, 256, 16 | 1 << 16),
    "tiles of 128 rows": (1100, 4128, 256, 256, 128 | 1 << 16), "pairs": (130, 13728, 224, 224, 0), "any distance": (40, 96, 77, 77, None),
}


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("name", PRODUCTS)
def test_products_in_8_bits_keep_nan(name, grouped):
    """A row and a column with NaN, under every epilogue: they and nothing else are NaN, the others as without them."""
    M, N, K_, apart, form = PRODUCTS[name]
    if form is not None and K().sm_count() == 148:
        assert K().lib().leb_linear_e4m3_form(1, M, N, K_, 148) == form
    x, xv = whole_numbers(M, K_, 1, apart)
    w, wv = whole_numbers(N, K_, 2, apart)
    sx, sw = powers(M, 4) / 64, powers(N, 3) / 16
    z = (xv @ wv.T) * sx.double()[:, None] * sw.double()
    row, gate, up = M // 2, 7, 32 + 16 + 5                      # column 7 is a gate, column 53 an up value
    sx[row], sw[gate], sw[up] = NAN, NAN, NAN
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[row], bad[:, gate], bad[:, up] = True, True, True
    off = torch.tensor([0, M], dtype=torch.int32, device=DEV) if grouped else None
    if grouped:
        args = (x, sx.to(DEV), torch.as_strided(w, (1, N, K_), (N * apart, apart, 1)), sw.to(DEV).view(1, N))
    else:
        args = (x, sx.to(DEV), w, sw.to(DEV))
    for dtype in (F32, BF16):
        half = 2.0 ** -8 if dtype is BF16 else 2.0 ** -24
        lost = bad.view(M, -1, 2, 16).any(2).reshape(M, -1)
        for act, code in gates().items():
            out = torch.zeros(M, N // 2, dtype=dtype, device=DEV)
            K().linear_e4m3(out, *args, code, group_offsets=off)
            got, want = out.cpu().double(), P.gated(z, act, 7.0)
            assert torch.equal(got.isnan(), lost), (act, dtype)
            b = z.view(M, -1, 2, 16)
            size = (b[:, :, 0].abs() * (b[:, :, 1].abs() + 1)).reshape(M, -1)
            unit = 2.0 ** -10 if dtype is BF16 and act == "gelu_tanh" else 2.0 ** -19      # (as where these epilogues are tested for their values)
            assert bool(((got - want).abs() <= half * 1.01 * want.abs() + unit * size + 1e-30)[~lost].all()), act
    for act, code in K().PLAIN_ACTIVATIONS.items():
        out = torch.zeros(M, N, dtype=BF16, device=DEV)
        K().linear_e4m3(out, *args, K().plain_act_epilogue(code), group_offsets=off)
        got, want = out.cpu().double(), P.PLAIN[act](z)
        assert torch.equal(got.isnan(), bad), act
        if act != "relu_squared":      # (z is exact; a square has no slope of at most 1.13)
            assert bool(((got - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + act_bound(z, 0.0))[~bad].all()), act
    K().check_device_status()


@pytest.mark.parametrize("M", [1, 8, 40, 130, 600])
def test_products_in_bfloat16_keep_nan(M):
    """The same epilogues behind the bfloat16 products, dense and grouped."""
    N, K_ = 320, 256
    k = K()
    x, w = gen(M, K_, seed=1, dtype=BF16).to(DEV), gen(N, K_, seed=2, scale=K_ ** -0.5, dtype=BF16).to(DEV)
    row = M // 2
    clean = {}
    off = torch.tensor([0, M], dtype=torch.int32, device=DEV)
    for turn in range(2):
        for kind, codes, width in (("gated", gates(), N // 2), ("plain", {a: k.plain_act_epilogue(c) for a, c in k.PLAIN_ACTIVATIONS.items()}, N)):
            for act, code in codes.items():
                for groups in (None, off):
                    out = torch.zeros(M, width, dtype=BF16, device=DEV)
                    k.linear(out, x, w if groups is None else w[None], code, group_offsets=groups)
                    if turn == 0:
                        clean[kind, act, groups is None] = out
                        assert bool(out.isfinite().all())
                        continue
                    assert bool(out[row].isnan().all()), (kind, act, groups)
                    rest = torch.arange(M, device=DEV) != row
                    assert torch.equal(out[rest], clean[kind, act, groups is None][rest])
        x[row, 3] = NAN
    k.check_device_status()


@pytest.mark.parametrize("M,F", [(1, 1), (3, 17), (9, 256)])
def test_activations_keep_nan(M, F):
    k = K()
    gu = gen(M, 2 * F, seed=1, scale=4.0)
    for bad in (0, F, 2 * F - 1):                               # a gate, an up value, the last
        v = gu.clone()
        v[M // 2, bad] = NAN
        lost = torch.zeros(M, F, dtype=torch.bool)
        lost[M // 2, bad % F] = True
        for dtype in (F32, BF16):
            for act in (k.SILU, k.GELU_TANH, k.CLAMPED_SIGMOID):
                for given in (F32, BF16) if dtype is BF16 else (F32,):
                    out, clean = torch.zeros(M, F, dtype=dtype, device=DEV), torch.zeros(M, F, dtype=dtype, device=DEV)
                    k.gated_act(out, v.to(given).to(DEV), act, 7.0, 1.5)
                    k.gated_act(clean, gu.to(given).to(DEV), act, 7.0, 1.5)
                    assert torch.equal(out.cpu().isnan(), lost) and torch.equal(out.cpu()[~lost], clean.cpu()[~lost])
            z = gu[:, :F].contiguous()
            zbad = z.clone()
            zbad[M // 2, bad % F] = NAN
            for code in k.PLAIN_ACTIVATIONS.values():
                out, clean = torch.zeros(M, F, dtype=dtype, device=DEV), torch.zeros(M, F, dtype=dtype, device=DEV)
                k.activation(out, zbad.to(DEV), code)
                k.activation(clean, z.to(DEV), code)
                assert torch.equal(out.cpu().isnan(), lost) and torch.equal(out.cpu()[~lost], clean.cpu()[~lost])
