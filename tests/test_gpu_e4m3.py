"""Products in 8 bits: rows brought to 8 bits, products of such rows, dense and grouped, and a run of them together, against the
definitions in double precision."""
import math

import pytest
import torch

import harness as H  # noqa: F401  (path setup)
import plain_e4m3 as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
NAN = float("nan")


def K():
    from lastengine_b200.ops import kernels
    return kernels


def gen(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype)


def room(M, width, pitch, dtype, fill=0):
    """[M, width] of rows `pitch` apart, all of it (what lies between the rows too) of one value; and the whole of it."""
    whole = torch.full((M * pitch + 64,), fill, dtype=torch.uint8 if dtype is E4M3 else dtype, device=DEV)
    whole = whole.view(dtype) if dtype is E4M3 else whole
    return torch.as_strided(whole, (M, width), (pitch, 1)), whole


def between(whole, M, width, pitch):
    """What lies between the rows of `room` and behind the last."""
    flat = whole.view(torch.uint8) if whole.dtype is E4M3 else whole
    return torch.cat([flat[:M * pitch].view(M, pitch)[:, width:].reshape(-1), flat[M * pitch:]])


# Rounded to float: 448 / a and the product with it, so a number is off by a factor of up to (1 + 2^-24)^2 before it is rounded
# to 8 bits; the norm's g = x w is one float product, made the same way here.
SLACK = 2.0 ** -22


def check_rows(q, scale, g, factor=None, scale_bound=2.0 ** -23):
    s, lo, hi = P.quantized(g.double(), SLACK)
    got = q.cpu().float().double()
    assert bool(((got >= lo) & (got <= hi)).all())
    want = s if factor is None else s * factor
    assert bool(((scale.cpu().double() - want).abs() <= scale_bound * want.abs()).all())


# ---- rows ------------------------------------------------------------------------------------------------------------
def test_the_format():
    """torch's type is the format of the definitions, so that what the kernels leave can be read through it."""
    v = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
    assert torch.equal(v, P.codes())
    x = gen(20000, seed=1, scale=40.0).double()
    assert torch.equal(x.to(F32).to(E4M3).double(), P.rounded(x.to(F32).double()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,D", [(1, 1), (3, 7), (5, 64), (2, 100), (7, 1000), (300, 1001), (1, 2048), (33, 2048), (9, 4096), (4, 8192),
                                 (13, 250), (21, 512), (9, 520), (6, 600), (3, 2500), (3, 3996), (2, 6001), (2, 8200), (2, 12001), (1, 16384), (3, 20000), (2, 50000)])
def test_quantize(dtype, M, D):
    x = gen(M, D, seed=M + D, dtype=dtype) * torch.exp(gen(M, 1, seed=3, scale=3.0)).to(dtype)
    for pitch_x, pitch_q in ((D, D), (D + 8, -(-D // 16) * 16), (D + 3, D + 5)):
        xd, _ = room(M, D, pitch_x, dtype)
        xd.copy_(x)
        q, whole = room(M, D, pitch_q, E4M3, 77)
        s = torch.empty(M, device=DEV)
        K().quantize_e4m3(q, s, xd)
        check_rows(q, s, x)
        assert bool((between(whole, M, D, pitch_q) == 77).all())


@pytest.mark.parametrize("D", [64, 1001, 2048])
def test_quantize_borders(D):
    """Ties, numbers below the least normal one, zeros, rows of zeros, rows too small for a scale, one number a row."""
    x = torch.zeros(8, D)
    x[0, :16] = torch.tensor([448.0, 17.0, 19.0, 18.0, -17.0, 0.001953125, 0.0009765625, 0.00146484375, 0.0029296875, 464.0 / 448, 1.0625, 1.1875, -0.0, 240.0, 248.0, 232.0])
    x[2, 5] = -3.0
    x[3] = 1e-33                       # below 2^-100: 448 x / 2^-100
    x[4, 0], x[4, 1] = 3e38, -1e38
    x[5, 0], x[5, 1] = 1e-40, -5e-41
    x[6] = 2.0 ** -100
    q, s = K().e4m3_rows(8, D, device=DEV), torch.empty(8, device=DEV)
    K().quantize_e4m3(q, s, x.to(DEV))
    check_rows(q, s, x)
    assert torch.equal(q[0, :16].cpu().double(), P.rounded(x[0, :16].double()))      # a = 448: nothing is scaled, ties to even
    assert torch.equal(q[1].cpu().float(), torch.zeros(D)) and float(s[1]) == float(torch.tensor(2.0 ** -100 / 448, dtype=F32))


@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("D", [40, 1001, 2048])
def test_rows_that_are_not_finite(bad, D):
    for at in (0, D - 1, D // 2):
        x = gen(3, D, seed=at)
        clean = x.clone()
        x[1, at] = bad
        for dtype in (F32, BF16):
            q, s = K().e4m3_rows(3, D, device=DEV), torch.zeros(3, device=DEV)
            K().quantize_e4m3(q, s, x.to(dtype).to(DEV))
            assert bool(q[1].float().isnan().all()) and bool(s[1].isnan())
            check_rows(q[::2], s[::2], clean.to(dtype)[::2])
        q, s = K().e4m3_rows(3, D, device=DEV), torch.zeros(3, device=DEV)
        K().rmsnorm_e4m3(q, s, x.to(DEV), torch.ones(D, device=DEV), 1e-5)
        assert bool(q[1].float().isnan().all()) and bool(s[1].isnan()) and not bool(s[::2].isnan().any())
        assert not bool(q[::2].float().isnan().any())


def test_squares_beyond_32_bits_are_no_norm():
    x = gen(2, 96, seed=1)
    x[1, 3] = 1e20
    q, s = K().e4m3_rows(2, 96, device=DEV), torch.zeros(2, device=DEV)
    K().rmsnorm_e4m3(q, s, x.to(DEV), torch.ones(96, device=DEV), 1e-5)
    assert bool(s[1].isnan()) and not bool(s[0].isnan())


@pytest.mark.parametrize("D", [64, 1001, 2048])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_gathered(D, dtype):
    """Rows in any order, some twice, some never, some that are not there; weights into the scales."""
    M, k = 11, 3
    x = gen(M, D, seed=5, dtype=dtype)
    rows = torch.tensor([32, 0, 0, 31, 7, 33, -1, 2 ** 31 - 1, 14, 14, 5, -2 ** 31], dtype=torch.int32)
    there = (rows >= 0) & (rows < M * k)
    weights = gen(M * k, seed=6)
    for w in (None, weights):
        q, s = K().e4m3_rows(len(rows), D, device=DEV), torch.zeros(len(rows), device=DEV)
        K().quantize_e4m3(q, s, x.to(DEV), rows=rows.to(DEV), div=k, weights=None if w is None else w.to(DEV))
        at = rows[there].long()
        check_rows(q.cpu().float()[there], s.cpu()[there], x[at // k], None if w is None else w.double()[at])
        assert bool(q.cpu().float()[~there].isnan().all()) and bool(s.cpu()[~there].isnan().all())


@pytest.mark.parametrize("y_dtype", [None, F32, BF16])
@pytest.mark.parametrize("M,D", [(1, 1), (2, 24), (5, 64), (7, 1000), (64, 1001), (1, 2048), (33, 2048), (3, 4096), (2, 8192),
                                 (13, 250), (21, 256), (9, 520), (3, 2500), (3, 3996), (2, 6001), (2, 8200), (2, 12001), (1, 16384), (2, 20000), (2000, 512)])
def test_rmsnorm(y_dtype, M, D):
    eps = 1e-5
    x, w = gen(M, D, seed=1, scale=2.0), 1 + 0.2 * gen(D, seed=2)
    y = None if y_dtype is None else gen(M, D, seed=3, dtype=y_dtype)
    for h_dtype in (None, F32, BF16):
        xd = x.to(DEV)
        pitch = -(-D // 16) * 16 if h_dtype is not F32 else D + 3
        q, whole = room(M, D, pitch, E4M3, 77)
        s, h = torch.empty(M, device=DEV), None if h_dtype is None else torch.empty(M, D, dtype=h_dtype, device=DEV)
        K().rmsnorm_e4m3(q, s, xd, w.to(DEV), eps, y=None if y is None else y.to(DEV), h=h)
        new = x if y is None else x + y.float()
        assert torch.equal(xd.cpu(), new)                                # one float addition
        r = 1 / torch.sqrt((new.double() ** 2).mean(1) + eps)
        # a thread's squares in order (the fewest threads are 32), then a tree: each sum is off by at most (D / 32 + 16) roundings,
        # the root halves that; mean, root, quotient and the two products of the scale round once each
        bound = 2.0 ** -24 * ((D / 32 + 16) / 2 + 6)
        g = new * w
        check_rows(q, s, g, r, bound)
        assert bool((between(whole, M, D, pitch) == 77).all())
        if h is not None:
            want = g.double() * r[:, None]
            step = 2.0 ** -8 if h_dtype is BF16 else 0.0
            assert bool(((h.cpu().double() - want).abs() <= (bound + step) * 1.01 * want.abs() + 1e-45).all())


@pytest.mark.parametrize("D", [250, 256, 501, 512, 1000, 1001, 1999, 2048, 3999, 4000, 6001, 8192, 8200, 12000, 16390])
def test_many_rows(D):
    """Rows enough to be shared out in the other way, few threads a row: the last block's are part of one."""
    M = 1029
    x, w, y = gen(M, D, seed=1, scale=2.0), 1 + 0.2 * gen(D, seed=2), gen(M, D, seed=3, dtype=BF16)
    for pitch in (-(-D // 16) * 16, D + 3):
        for t in (x, y):
            q, whole = room(M, D, pitch, E4M3, 77)
            s = torch.empty(M, device=DEV)
            K().quantize_e4m3(q, s, t.to(DEV))
            check_rows(q, s, t)
            assert bool((between(whole, M, D, pitch) == 77).all())
        for added in (None, y, y.float()):
            q, whole = room(M, D, pitch, E4M3, 77)
            s, xd, h = torch.empty(M, device=DEV), x.to(DEV), torch.empty(M, D, device=DEV)
            K().rmsnorm_e4m3(q, s, xd, w.to(DEV), 1e-5, y=None if added is None else added.to(DEV), h=h)
            new = x if added is None else x + y.float()
            assert torch.equal(xd.cpu(), new)
            r = 1 / torch.sqrt((new.double() ** 2).mean(1) + 1e-5)
            bound = 2.0 ** -24 * ((D / 32 + 16) / 2 + 6)                 # (as above)
            check_rows(q, s, new * w, r, bound)
            want = (new * w).double() * r[:, None]
            assert bool(((h.cpu().double() - want).abs() <= bound * 1.01 * want.abs() + 1e-45).all())
            assert bool((between(whole, M, D, pitch) == 77).all())


def test_no_rows():
    q, s = K().e4m3_rows(0, 64, device=DEV), torch.empty(0, device=DEV)
    K().quantize_e4m3(q, s, torch.empty(0, 64, device=DEV))
    K().rmsnorm_e4m3(q, s, torch.empty(0, 64, device=DEV), torch.ones(64, device=DEV), 1e-5)
    w, sw = torch.zeros(32, 64, device=DEV).to(E4M3), torch.ones(32, device=DEV)
    K().linear_e4m3(torch.empty(0, 32, device=DEV), q, s, w, sw)


# ---- products --------------------------------------------------------------------------------------------------------
def whole_numbers(M, K_, seed, pitch=None):
    """Whole numbers from -8 to 8 in 8 bits (all held exactly), rows `pitch` apart with NaN between them; and as doubles."""
    v = torch.randint(-8, 9, (M, K_), generator=torch.Generator().manual_seed(seed)).float()
    pitch = pitch or -(-K_ // 16) * 16
    q, _ = room(M, K_, pitch, E4M3, 0x7f)
    q.copy_(v.to(E4M3))
    return q, v.double()


def powers(n, seed):
    return 2.0 ** torch.randint(-3, 4, (n,), generator=torch.Generator().manual_seed(seed)).float()


ROWS = [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 200, 256, 257, 500, 1025]
SIZES = [(32, 16), (1, 1), (17, 128), (96, 100), (128, 129), (160, 256), (130, 1000), (300, 2048), (2080, 640), (513, 4100), (64, 9000)]


@pytest.mark.parametrize("N,K_", SIZES)
@pytest.mark.parametrize("pitch", [16, 1])
def test_linear_is_exact_on_whole_numbers(N, K_, pitch):
    """Every sum is a whole number below 2^24 and every scale a power of two, so that the float result is exact whatever the order of
    the sums: any row, column or number of k left out, taken twice or misplaced shows.  Rows 16 bytes apart, and an odd number."""
    apart = -(-K_ // 16) * 16 if pitch == 16 else (K_ + 1) | 1
    w, wv = whole_numbers(N, K_, 2, apart)
    sw = powers(N, 3)
    for M in ROWS if pitch == 16 else (1, 17, 130):
        x, xv = whole_numbers(M, K_, M, apart)
        sx = powers(M, 4)
        z = (xv @ wv.T) * sx.double()[:, None] * sw.double()
        for ldc in (N, N + 5):
            out, whole = room(M, N, ldc, F32, 5)
            K().linear_e4m3(out, x, sx.to(DEV), w, sw.to(DEV))
            assert torch.equal(out.cpu().double(), z), (M, N, K_)
            K().linear_e4m3(out, x, sx.to(DEV), w, sw.to(DEV), K().ACCUMULATE)
            assert torch.equal(out.cpu().double(), 2 * z), (M, N, K_)
            assert bool((between(whole, M, N, ldc) == 5).all())
        out, whole = room(M, N, N + 8, BF16, 5)
        K().linear_e4m3(out, x, sx.to(DEV), w, sw.to(DEV))
        assert torch.equal(out.cpu(), z.float().to(BF16)), (M, N, K_)
        assert bool((between(whole, M, N, N + 8) == 5).all())
    K().check_device_status()


def act_bound(z, dz):
    """How far an activation of slope at most 1.13 (times up, of slope 1) of values off by dz may be, with its own eight float roundings of
    2^-24 and the special function unit's 2^-20."""
    return 1.2 * dz + 2.0 ** -19 * z.abs() + 1e-30


@pytest.mark.parametrize("M", [1, 16, 33, 128, 129, 300, 1100])
@pytest.mark.parametrize("N,K_,apart", [(64, 64, 64), (320, 1000, 1008), (4128, 256, 256), (96, 77, 77)])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_linear_gated_and_activated(M, N, K_, apart, out_dtype):
    x, xv = whole_numbers(M, K_, M, apart)
    w, wv = whole_numbers(N, K_, 2, apart)
    sx, sw = powers(M, 4) / 64, powers(N, 3) / 16
    z = (xv @ wv.T) * sx.double()[:, None] * sw.double()      # exact in float: what differs is the activation's own arithmetic
    half = 2.0 ** -8 if out_dtype is BF16 else 2.0 ** -24
    for name, code in (("silu", K().gated_epilogue(K().SILU)), ("gelu_tanh", K().gated_epilogue(K().GELU_TANH)), ("clamped", K().gated_epilogue(K().CLAMPED_SIGMOID, 7.0, 1.702))):
        out, whole = room(M, N // 2, N // 2 + 8, out_dtype, 5)
        K().linear_e4m3(out, x, sx.to(DEV), w, sw.to(DEV), code)
        want = P.gated(z, name, 7.0)
        up = z.reshape(M, -1, 2, 16)
        size = (up[:, :, 0].abs() * (up[:, :, 1].abs() + 1)).reshape(M, -1)       # |gate| (|up| + 1): what relative errors of the factors go by
        # gelu's tanh comes from the special function unit for bfloat16 results (2^-10.9 of 1 + tanh's magnitude)
        unit = 2.0 ** -10 if out_dtype is BF16 and name == "gelu_tanh" else 2.0 ** -19
        assert bool(((out.cpu().double() - want).abs() <= half * 1.01 * want.abs() + unit * size + 1e-30).all()), name
        assert bool((between(whole, M, N // 2, N // 2 + 8) == 5).all())
    if out_dtype is BF16:
        for name, code in K().PLAIN_ACTIVATIONS.items():
            out, whole = room(M, N, N + 8, out_dtype, 5)
            K().linear_e4m3(out, x, sx.to(DEV), w, sw.to(DEV), K().plain_act_epilogue(code))
            want = P.PLAIN[name](z)
            assert bool(((out.cpu().double() - want).abs() <= half * 1.01 * want.abs() + 2.0 ** -19 * z.abs() + 1e-30).all()), name
            assert bool((between(whole, M, N, N + 8) == 5).all())
    K().check_device_status()


@pytest.mark.parametrize("M,N,K_", [(1, 512, 2048), (40, 300, 4096), (130, 256, 8192), (700, 2048, 2048), (2048, 4096, 1024), (3, 64, 12000)])
def test_linear_sums(M, N, K_):
    """Numbers of all sizes.  An element's sum of n products in float is off by at most n 2^-23 of the sum of their magnitudes (a
    tensor core cuts, it does not round); over all elements the errors' signs differ or they are shared out over the row, and the norm of
    the differences is held to 2^-20 of the result's: an accumulator of fewer than 24 bits would not pass."""
    x, sx = K().e4m3_rows(M, K_, device=DEV), torch.empty(M, device=DEV)
    w, sw = K().e4m3_rows(N, K_, device=DEV), torch.empty(N, device=DEV)
    K().quantize_e4m3(x, sx, gen(M, K_, seed=1).to(DEV))
    K().quantize_e4m3(w, sw, gen(N, K_, seed=2).to(DEV))
    z, size = P.product(x.cpu(), sx.cpu(), w.cpu(), sw.cpu())
    out = torch.empty(M, N, device=DEV)
    K().linear_e4m3(out, x, sx, w, sw)
    d = (out.cpu().double() - z).abs()
    assert bool((d <= (K_ + 4) * 2.0 ** -23 * size).all())
    assert float(d.norm() / z.norm()) < 2.0 ** -20
    again = torch.empty(M, N, device=DEV)
    K().linear_e4m3(again, x, sx, w, sw)
    assert torch.equal(out, again)
    K().check_device_status()


def test_rows_apart_from_one_another():
    """A row that is not finite (its scale is NaN) makes its own results NaN and no other's; so does a weight row."""
    M, N, K_ = 40, 96, 256
    for rows in (1, 20, 40, 200, 1100):
        x, sx = whole_numbers(rows, K_, 1)[0], torch.ones(rows)
        w, sw = whole_numbers(N, K_, 2)[0], torch.ones(N)
        want = torch.empty(rows, N, device=DEV)
        K().linear_e4m3(want, x, sx.to(DEV), w, sw.to(DEV))
        sx[rows // 2], sw[7] = NAN, NAN
        x[rows // 2] = torch.full((K_,), NAN, device=DEV).to(E4M3)
        out = torch.empty(rows, N, device=DEV)
        K().linear_e4m3(out, x, sx.to(DEV), w, sw.to(DEV))
        nan = torch.zeros(rows, N, dtype=torch.bool, device=DEV)
        nan[rows // 2], nan[:, 7] = True, True
        assert bool(out[nan].isnan().all()) and torch.equal(out[~nan], want[~nan])


GROUPS = [
    [0, 0, 0, 0], [1], [5], [0, 3, 0], [16, 17, 1, 0, 33, 2], [130, 0, 1, 64, 7], [300, 20, 0, 0, 513], [1] * 40, [4] * 256, [0] * 255 + [9], [700], [1200, 1, 900],
]


@pytest.mark.parametrize("counts", GROUPS, ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("N,K_,apart", [(32, 16, 16), (200, 300, 304), (384, 1000, 1008), (65, 30, 31)])
def test_grouped_is_exact_on_whole_numbers(counts, N, K_, apart):
    E, behind = len(counts), 5
    total = sum(counts)
    M = total + behind
    x, xv = whole_numbers(M, K_, 1, apart)
    w2, wv = whole_numbers(E * N, K_, 2, apart)
    w = torch.as_strided(w2, (E, N, K_), (N * apart, apart, 1))
    sx, sw = powers(M, 4), powers(E * N, 3).view(E, N)
    off = torch.tensor([sum(counts[:e]) for e in range(E + 1)], dtype=torch.int32)
    z, _ = P.product(xv, sx, wv.view(E, N, K_), sw, off)
    for dtype in (F32, BF16):
        out, whole = room(M, N, N + 3, dtype, 5)
        K().linear_e4m3(out, x, sx.to(DEV), w, sw.to(DEV), group_offsets=off.to(DEV))
        assert torch.equal(out[:total].cpu(), z[:total].float().to(dtype))
        assert bool((out[total:] == 5).all()) and bool((between(whole, M, N, N + 3) == 5).all())
    out, whole = room(M, N, N, F32, 5)
    K().linear_e4m3(out, x, sx.to(DEV), w, sw.to(DEV), K().ACCUMULATE, group_offsets=off.to(DEV))
    assert torch.equal(out[:total].cpu().double(), z[:total] + 5) and bool((out[total:] == 5).all())
    if N % 32 == 0:
        small = sx / 64
        out, whole = room(M, N // 2, N // 2, BF16, 5)
        K().linear_e4m3(out, x, small.to(DEV), w, sw.to(DEV), K().gated_epilogue(K().SILU), group_offsets=off.to(DEV))
        zs = z / 64
        want = P.gated(zs, "silu")
        up = zs.reshape(M, -1, 2, 16)
        size = (up[:, :, 0].abs() * up[:, :, 1].abs()).reshape(M, -1)
        d = (out.cpu().double() - want).abs()[:total]
        assert bool((d <= 2.0 ** -8 * 1.01 * want.abs()[:total] + 2.0 ** -19 * size[:total] + 1e-30).all())
        assert bool((out[total:] == 5).all())
    K().check_device_status()


# (groups, rows of each, columns, K) by the form that takes them on 148 SMs: rows of a tile and slices of K (64 rows: with fewer tiles than SMs
# and with more), or pairs
FORMS = {
    "16, 1": (1, 1, 151, 211), "16, 2": (1, 1, 150, 664), "16, 4": (1, 1, 154, 904), "16, 8": (1, 1, 154, 1921),
    "32, 1": (1, 132, 150, 205), "32, 2": (1, 18, 9654, 4090), "32, 4": (1, 17, 1169, 929), "32, 8": (1, 17, 523, 2113),
    "64, 1": (1, 783, 150, 222), "64, 1, many": (1, 33, 19777, 203), "64, 4": (1, 33, 2397, 1492), "64, 8": (1, 34, 1353, 1978),
    "128, 1": (1, 65, 7455, 202), "pairs": (1, 139, 13706, 213), "pairs, results that copies take": (1, 139, 13712, 208),
}
GROUPED_FORMS = {
    "16, 1": (2, 1, 171, 213), "16, 2": (2, 1, 151, 646), "16, 4": (2, 1, 157, 951), "16, 8": (2, 1, 167, 2087),
    "32, 1": (15, 17, 167, 203), "32, 2": (5, 17, 1849, 3559), "32, 4": (6, 17, 154, 1165), "32, 8": (2, 18, 354, 2058),
    "64, 1": (28, 34, 156, 212), "64, 1, many": (59, 33, 266, 200), "64, 4": (9, 34, 203, 1829), "64, 8": (6, 33, 196, 2109),
    "128, 1": (20, 65, 275, 262), "pairs": (56, 155, 178, 217), "pairs, results that copies take": (56, 155, 192, 224),
}


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_every_form_is_exact_on_whole_numbers(form, grouped):
    """Each kernel, tile and way to cut K, at sizes that nothing divides: stored, added, gated, activated, in both types, rows that TMA stores
    and rows that it does not."""
    E, r, N, K_ = (GROUPED_FORMS if grouped else FORMS)[form]
    sms = K().sm_count()
    got = K().lib().leb_linear_e4m3_form(E, r, N, K_, sms)
    if sms == 148:
        assert got == (0 if form.startswith("pairs") else int(form.split(", ")[0]) | int(form.split(", ")[1]) << 16)
        if form.startswith("64, 1"):
            assert (E * -(-r // 64) * -(-N // 128) <= sms) == (form == "64, 1")
    M = E * r
    counts = [r] * E
    if grouped and E > 2:              # as many rows in all, shared out unevenly
        counts[0], counts[1], counts[-1] = 0, counts[1] + (r + 1) // 2, counts[-1] + r // 2
    off = torch.tensor([sum(counts[:e]) for e in range(E + 1)], dtype=torch.int32, device=DEV) if grouped else None
    apart = -(-K_ // 16) * 16
    x, xv = whole_numbers(M, K_, 1, apart)
    w, wv = whole_numbers(E * N, K_, 2, apart)
    sx, sw = powers(M, 4).to(DEV), powers(E * N, 3).to(DEV)
    xd, wd = xv.to(DEV) * sx.double()[:, None], wv.to(DEV) * sw.double()[:, None]
    z = torch.cat([xd[sum(counts[:e]):sum(counts[:e + 1])] @ wd[e * N:(e + 1) * N].T for e in range(E)]) if grouped else xd @ wd.T
    args = (x, sx, torch.as_strided(w, (E, N, K_), (N * apart, apart, 1)), sw.view(E, N)) if grouped else (x, sx, w, sw)
    for ldc in (-(-N // 8) * 8, N):
        out, whole = room(M, N, ldc, F32, 5)
        K().linear_e4m3(out, *args, group_offsets=off)
        assert torch.equal(out.double(), z)
        K().linear_e4m3(out, *args, K().ACCUMULATE, group_offsets=off)
        assert torch.equal(out.double(), 2 * z) and bool((between(whole, M, N, ldc) == 5).all())
        out, whole = room(M, N, ldc, BF16, 5)
        K().linear_e4m3(out, *args, group_offsets=off)
        assert torch.equal(out, z.float().to(BF16)) and bool((between(whole, M, N, ldc) == 5).all())
        K().linear_e4m3(out, *args, K().plain_act_epilogue(K().PLAIN_ACTIVATIONS["relu_squared"]), group_offsets=off)
        # (a square of up to 2^21 is rounded to float once, and to bfloat16)
        want = z.clamp(min=0) ** 2
        assert bool(((out.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -24) * 1.01 * want).all())
    n = N // 32 * 32                   # gated: whole blocks of 32 rows of every expert's weights
    w3 = torch.as_strided(w, (E, n, K_), (n * apart, apart, 1)) if grouped else w[:n]
    wv3 = wv.to(DEV).reshape(-1)[:E * n * K_].view(E, n, K_)
    s3 = sw[:E * n] / 1024
    z3 = torch.cat([xd[sum(counts[:e]):sum(counts[:e + 1])] @ (wv3[e] * s3[e * n:(e + 1) * n].double()[:, None]).T for e in range(E)]) if grouped else xd @ (wv3[0] * s3.double()[:, None]).T
    want, b = P.gated(z3, "silu"), z3.reshape(M, -1, 2, 16)
    size = (b[:, :, 0].abs() * b[:, :, 1].abs()).reshape(M, -1)
    for dtype in (F32, BF16):
        for ldc in (n // 2, n // 2 + 1):
            out, whole = room(M, n // 2, ldc, dtype, 5)
            K().linear_e4m3(out, x, sx, w3, s3.view(E, n) if grouped else s3, K().gated_epilogue(K().SILU), group_offsets=off)
            half = 2.0 ** -8 if dtype is BF16 else 2.0 ** -24
            assert bool(((out.double() - want).abs() <= half * 1.01 * want.abs() + 2.0 ** -19 * size + 1e-30).all())
            assert bool((between(whole, M, n // 2, ldc) == 5).all())
    K().check_device_status()


@pytest.mark.parametrize("pitch", [16, 1])
def test_offsets_that_are_not_in_order_touch_nothing_else(pitch):
    """Offsets that fall, are negative or go beyond the rows: a row gets numbers of an expert or stays, nothing beyond out is written."""
    E, N, K_ = 4, 96, 64
    apart = 64 if pitch == 16 else 65
    for M, k in ((50, 1), (3000, 60)):
        x, xv = whole_numbers(M, K_, 1, apart)
        wq, wv = whole_numbers(E * N, K_, 2, apart)
        w = torch.as_strided(wq, (E, N, K_), (N * apart, apart, 1))
        one, sw = torch.ones(M, device=DEV), torch.ones(E, N, device=DEV)
        z = torch.stack([xv @ wv[e * N:(e + 1) * N].T for e in range(E)]).to(DEV)
        for off in ([0, 40, 10, 60, 2 ** 31 - 1], [-5, 10, 20, 30, 40], [50, 40, 30, 20, 10], [-2 ** 31, 2 ** 31 - 1, 0, 0, 0], [0, 50, 0, 50, 0]):
            off = [o * k if abs(o) < 1000 else o for o in off]
            out, whole = room(M, N, N + 3, F32, 0.5)
            K().linear_e4m3(out, x, one, w, sw, group_offsets=torch.tensor(off, dtype=torch.int32, device=DEV))
            assert bool((between(whole, M, N, N + 3) == 0.5).all())
            row_is = torch.stack([(out.double() == z[e]).all(1) for e in range(E)] + [(out == 0.5).all(1)]).any(0)
            assert bool(row_is.all())
    K().check_device_status()


def test_weights_made_right_before():
    """Weights and rows that the launches right before write: the product waits for them."""
    N, K_ = 4096, 2048
    w, sw = K().e4m3_rows(N, K_, device=DEV), torch.zeros(N, device=DEV)
    x, sx = K().e4m3_rows(8, K_, device=DEV), torch.zeros(8, device=DEV)
    outs = []
    for turn in range(6):
        wf, xf = gen(N, K_, seed=turn % 2).to(DEV), gen(8, K_, seed=7).to(DEV)
        out = torch.empty(8, N, device=DEV)
        K().quantize_e4m3(x, sx, xf)
        K().quantize_e4m3(w, sw, wf)
        K().linear_e4m3(out, x, sx, w, sw)
        outs.append(out)
    z, size = P.product(x.cpu(), sx.cpu(), w.cpu(), sw.cpu())
    assert torch.equal(outs[5], outs[1]) and torch.equal(outs[4], outs[0]) and not torch.equal(outs[5], outs[4])
    assert float((outs[5].cpu().double() - z).norm() / z.norm()) < 2.0 ** -20


def test_places_beyond_32_bits():
    """Results, rows and 8-bit numbers of more than 2^31 numbers: the last rows are where they belong, and right."""
    M, N, K_ = 33000, 66016, 64
    x, xv = whole_numbers(M, K_, 1)
    w, wv = whole_numbers(N, K_, 2)
    out = torch.zeros(M, N, dtype=BF16, device=DEV)
    K().linear_e4m3(out, x, torch.ones(M, device=DEV), w, torch.ones(N, device=DEV))
    at = [0, 1, 16383, 32767, 32768, M - 1]
    assert torch.equal(out[at].double().cpu(), (xv[at] @ wv.T).float().to(BF16).double())
    q, s = K().e4m3_rows(M, N, device=DEV), torch.zeros(M, device=DEV)
    K().quantize_e4m3(q, s, out)
    check_rows(q[at], s[at], out[at].cpu())
    del out, q
    M, D = 265000, 8192
    xs = torch.ones(M, D, device=DEV)
    xs[at] = gen(len(at), D, seed=3).to(DEV)
    xs[-1] = gen(D, seed=4).to(DEV)
    at.append(M - 1)
    keep = xs[at].cpu()
    q, s = K().e4m3_rows(M, D, device=DEV), torch.zeros(M, device=DEV)
    K().rmsnorm_e4m3(q, s, xs, torch.ones(D, device=DEV), 1e-5)
    r = 1 / torch.sqrt((keep.double() ** 2).mean(1) + 1e-5)
    check_rows(q[at], s[at], keep, r, 2.0 ** -24 * ((D / 32 + 16) / 2 + 6))


# ---- together --------------------------------------------------------------------------------------------------------
def test_a_feed_forward_in_8_bits():
    """norm -> gate and up -> rows -> down into the stream, as a layer runs them; captured and replayed, and on a stream of its own."""
    M, D, F = 37, 256, 512
    x0, y, w = gen(M, D, seed=1, scale=2.0), gen(M, D, seed=2, dtype=BF16), 1 + 0.1 * gen(D, seed=3)
    w13, w2 = gen(2 * F, D, seed=4, scale=D ** -0.5), gen(D, F, seed=5, scale=F ** -0.5)
    k = K()
    dev = lambda t: t.to(DEV)  # noqa: E731
    q13, s13, q2, s2 = k.e4m3_rows(2 * F, D, device=DEV), torch.empty(2 * F, device=DEV), k.e4m3_rows(D, F, device=DEV), torch.empty(D, device=DEV)
    k.quantize_e4m3(q13, s13, dev(w13))
    k.quantize_e4m3(q2, s2, dev(w2))
    x, yd, wd = dev(x0), dev(y), dev(w)
    h8, hs, a, a8, as_ = k.e4m3_rows(M, D, device=DEV), torch.empty(M, device=DEV), torch.empty(M, F, dtype=BF16, device=DEV), k.e4m3_rows(M, F, device=DEV), torch.empty(M, device=DEV)

    def layer():
        k.rmsnorm_e4m3(h8, hs, x, wd, 1e-5, y=yd)
        k.linear_e4m3(a, h8, hs, q13, s13, k.gated_epilogue(k.SILU))
        k.quantize_e4m3(a8, as_, a)
        k.linear_e4m3(x, a8, as_, q2, s2, k.ACCUMULATE)

    layer()
    new = x0.double() + y.double()
    h = P.product(h8.cpu(), hs.cpu(), q13.cpu(), s13.cpu())[0]
    act = P.gated(h, "silu")
    assert float((a.cpu().double() - act).norm() / act.norm()) < 2.0 ** -8
    down = P.product(a8.cpu(), as_.cpu(), q2.cpu(), s2.cpu())[0]
    assert float((x.cpu().double() - new - down).norm() / x.cpu().double().norm()) < 2.0 ** -20
    # against the layer without 8 bits: each of the four roundings to 8 bits is half a step of 2^-4 at most, some 2.6% on average
    hf = new / torch.sqrt((new ** 2).mean(1, keepdim=True) + 1e-5) * w.double()
    want = P.gated(hf @ w13.double().T, "silu") @ w2.double().T
    assert float((down - want).norm() / want.norm()) < 4 * 2.0 ** -4
    first = x.clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.copy_(dev(x0))
        layer()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(x, first)
    with torch.cuda.graph(graph):
        layer()
    for _ in range(3):
        x.copy_(dev(x0))
        graph.replay()
        assert torch.equal(x, first)
    k.check_device_status()


def test_experts_in_8_bits():
    """router's choice -> rows in the experts' order -> the two grouped products -> their weighted sum."""
    M, D, F, E, kk = 70, 128, 96, 10, 3
    k = K()
    h, ids = gen(M, D, seed=1, dtype=BF16), torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(m))[:kk] for m in range(M)]).to(torch.int32)
    wts = torch.rand(M, kk, generator=torch.Generator().manual_seed(2))
    w13, w2 = gen(E * 2 * F, D, seed=4, scale=D ** -0.5), gen(E * D, F, seed=5, scale=F ** -0.5)
    q13, s13 = k.e4m3_rows(E * 2 * F, D, device=DEV), torch.empty(E * 2 * F, device=DEV)
    q2, s2 = k.e4m3_rows(E * D, F, device=DEV), torch.empty(E * D, device=DEV)
    k.quantize_e4m3(q13, s13, w13.to(DEV))
    k.quantize_e4m3(q2, s2, w2.to(DEV))
    PAIRS = M * kk
    word = lambda n: torch.empty(n, dtype=torch.int32, device=DEV)  # noqa: E731
    off, order, place = word(E + 1), word(PAIRS), word(PAIRS)
    hd, idd, wd = h.to(DEV), ids.to(DEV), wts.to(DEV)
    for weigh_input in (False, True):
        k.moe_align(off, order, place, idd, E)
        xs, ss = k.e4m3_rows(PAIRS, D, device=DEV), torch.empty(PAIRS, device=DEV)
        k.quantize_e4m3(xs, ss, hd, rows=order, div=kk, weights=wd.view(-1) if weigh_input else None)
        a, a8, as_ = torch.empty(PAIRS, F, dtype=BF16, device=DEV), k.e4m3_rows(PAIRS, F, device=DEV), torch.empty(PAIRS, device=DEV)
        k.linear_e4m3(a, xs, ss, q13.view(E, 2 * F, D), s13.view(E, 2 * F), k.gated_epilogue(k.SILU), group_offsets=off)
        k.quantize_e4m3(a8, as_, a)
        ys = torch.empty(PAIRS, D, device=DEV)
        k.linear_e4m3(ys, a8, as_, q2.view(E, D, F), s2.view(E, D), group_offsets=off)
        out = torch.zeros(M, D, device=DEV)
        k.moe_combine(out, ys, place, None if weigh_input else wd, False, k=kk)
        W13 = (q13.cpu().double() * s13.cpu().double()[:, None]).view(E, 2 * F, D)
        W2 = (q2.cpu().double() * s2.cpu().double()[:, None]).view(E, D, F)
        want = torch.zeros(M, D, dtype=torch.float64)
        for m in range(M):
            for j in range(kk):
                e, f = int(ids[m, j]), float(wts[m, j])
                z = P.gated((h[m].double() * (f if weigh_input else 1))[None] @ W13[e].T, "silu") @ W2[e].T
                want[m] += z[0] * (1 if weigh_input else f)
        # the rows' two roundings to 8 bits, half a step of 2^-4 each at most
        assert float((out.cpu().double() - want).norm() / want.norm()) < 2 * 2.0 ** -4
    k.check_device_status()
