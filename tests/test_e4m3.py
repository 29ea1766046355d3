"""Products in 8 bits, on the host: what the calls refuse before anything is launched, and what they hand on."""
import struct
import types

import pytest
import torch

import harness as H  # noqa: F401  (path setup)
import plain_e4m3 as P
from lastengine_b200.ops import kernels as K

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.fixture
def calls(monkeypatch):
    """The entry points' arguments, in the place of the entry points."""
    got = []

    def record(name, form):
        return lambda packed, stream: got.append((name, struct.unpack(form, packed))) or 0

    forms = {"leb_quantize_e4m3": "12q", "leb_rmsnorm_e4m3": "11qd", "leb_linear_e4m3": "17q"}
    monkeypatch.setattr(K, "lib", lambda: types.SimpleNamespace(**{n: record(n, f) for n, f in forms.items()}))
    monkeypatch.setattr(K, "_not_here", lambda *a, **k: None)
    monkeypatch.setattr(K, "_status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(K, "_stream_on", lambda device: 0)
    return got


def eight(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(E4M3)


def test_rounding_of_the_definition():
    """The format's own numbers stay, ties go to the even code, what is larger than 448 to 448."""
    v = P.codes()
    assert torch.equal(P.rounded(v), v) and torch.equal(P.rounded(-v), -v)
    mid = (v[1:] + v[:-1]) / 2
    even = torch.where(torch.arange(126) % 2 == 0, v[:-1], v[1:])
    assert torch.equal(P.rounded(mid), even) and float(P.rounded(torch.tensor([1e9], dtype=torch.float64))) == 448


def test_rows_16_bytes_apart():
    for k in (1, 15, 16, 17, 1001):
        t = K.e4m3_rows(3, 5, k)
        assert t.shape == (3, 5, k) and t.dtype == E4M3 and t.stride(1) % 16 == 0 and t.stride(1) - k < 16 and t.stride(0) == 5 * t.stride(1)


def test_cpu_tensors_are_refused():
    with pytest.raises(K.KernelError, match="CUDA"):
        K.quantize_e4m3(eight(2, 16), torch.zeros(2), torch.zeros(2, 16))
    with pytest.raises(K.KernelError, match="CUDA"):
        K.rmsnorm_e4m3(eight(2, 16), torch.zeros(2), torch.zeros(2, 16), torch.zeros(16), 1e-5)
    with pytest.raises(K.KernelError, match="CUDA"):
        K.linear_e4m3(torch.zeros(2, 3), eight(2, 16), torch.zeros(2), eight(3, 16), torch.zeros(3))


def test_another_device_is_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    there = types.SimpleNamespace(get_device=lambda: 0, device="cuda:0", is_cuda=True)
    with pytest.raises(K.KernelError, match="current device is cuda:1"):
        K._not_here("linear_e4m3", x=None, w=there)


def quantize(out=None, scale=None, x=None, **kw):
    K.quantize_e4m3(eight(4, 32) if out is None else out, torch.zeros(4) if scale is None else scale, torch.zeros(4, 32) if x is None else x, **kw)


def test_quantize_refusals(calls):
    rows = torch.zeros(4, dtype=torch.int32)
    for bad in (dict(out=torch.zeros(4, 32)), dict(out=eight(4, 31)), dict(out=eight(3, 32)), dict(out=eight(32, 4).t()), dict(out=eight(1, 32).expand(4, 32)), dict(out=eight(128)),
                dict(x=torch.zeros(4, 32, dtype=torch.float16)), dict(x=torch.zeros(32, 4).t()), dict(x=torch.zeros(128)), dict(x=torch.zeros(5, 32)),
                dict(scale=torch.zeros(5)), dict(scale=torch.zeros(4, dtype=BF16)), dict(scale=torch.zeros(8)[::2]), dict(scale=torch.zeros(4, 1)),
                dict(rows=rows.long()), dict(rows=rows[:3]), dict(rows=rows, div=0), dict(rows=rows, div=-1), dict(div=2), dict(weights=torch.zeros(4)),
                dict(rows=rows, weights=torch.zeros(3)), dict(rows=rows, div=2, weights=torch.zeros(7)), dict(rows=rows, weights=torch.zeros(4, dtype=BF16)),
                dict(x=torch.zeros(4, 0), out=eight(4, 0))):
        with pytest.raises(K.KernelError):
            quantize(**bad)
    assert not calls
    quantize(x=torch.zeros(2, 32), rows=rows, div=3, weights=torch.zeros(6))
    quantize(x=torch.zeros(1, 32).expand(4, 32))                       # one row four times: read, not written
    quantize(out=K.e4m3_rows(4, 30), x=torch.zeros(4, 30, dtype=BF16))
    K.quantize_e4m3(eight(0, 32), torch.zeros(0), torch.zeros(0, 32))
    assert [a[6:] for _, a in calls] == [(3, 4, 2, 32, 32, 32), (1, 4, 4, 32, 0, 32), (1, 4, 4, 30, 30, 32)]


def norm(out=None, scale=None, x=None, w=None, eps=1e-5, **kw):
    K.rmsnorm_e4m3(eight(4, 32) if out is None else out, torch.zeros(4) if scale is None else scale, torch.zeros(4, 32) if x is None else x,
                   torch.zeros(32) if w is None else w, eps, **kw)


def test_rmsnorm_refusals(calls):
    for bad in (dict(out=torch.zeros(4, 32)), dict(out=eight(4, 31)), dict(out=eight(1, 32).expand(4, 32)), dict(out=eight(32, 4).t()), dict(scale=torch.zeros(3)),
                dict(scale=torch.zeros(4, dtype=BF16)), dict(x=torch.zeros(4, 32, dtype=BF16)), dict(x=torch.zeros(4, 40)[:, :32]), dict(x=torch.zeros(128)),
                dict(w=torch.zeros(31)), dict(w=torch.zeros(32, dtype=BF16)), dict(y=torch.zeros(4, 31)), dict(y=torch.zeros(4, 40)[:, :32]),
                dict(y=torch.zeros(4, 32, dtype=torch.float16)), dict(h=torch.zeros(4, 32, dtype=torch.float16)), dict(h=torch.zeros(3, 32)), dict(h=torch.zeros(32, 4).t()),
                dict(x=torch.zeros(4, 0), out=eight(4, 0), w=torch.zeros(0))):
        with pytest.raises(K.KernelError):
            norm(**bad)
    assert not calls
    norm(y=torch.zeros(4, 32, dtype=BF16), h=torch.zeros(4, 32))
    norm(out=torch.as_strided(eight(200), (4, 32), (33, 1)))
    assert [(a[5], *a[7:]) for _, a in calls] == [(K.BF16, K.F32, 4, 32, 32, 1e-5), (K.F32, K.F32, 4, 32, 33, 1e-5)]


def linear(out=None, x=None, x_scale=None, w=None, w_scale=None, *a, **kw):
    K.linear_e4m3(torch.zeros(4, 64) if out is None else out, eight(4, 32) if x is None else x, torch.zeros(4) if x_scale is None else x_scale,
                  eight(64, 32) if w is None else w, torch.zeros(64) if w_scale is None else w_scale, *a, **kw)


def test_linear_refusals(calls):
    silu = K.gated_epilogue(K.SILU)
    for bad in (dict(out=torch.zeros(4, 63)), dict(out=torch.zeros(3, 64)), dict(out=torch.zeros(4, 64, dtype=torch.float16)), dict(out=torch.zeros(64, 4).t()),
                dict(out=torch.zeros(1, 64).expand(4, 64)), dict(out=torch.zeros(256)), dict(x=torch.zeros(4, 32)), dict(x=eight(4, 31)), dict(x=eight(32, 4).t()), dict(x=eight(128)),
                dict(x_scale=torch.zeros(3)), dict(x_scale=torch.zeros(4, 1)), dict(x_scale=torch.zeros(4, dtype=BF16)), dict(w=torch.zeros(64, 32)), dict(w=eight(64, 33)),
                dict(w=eight(32, 64).t()), dict(w=eight(1, 64, 32)), dict(w_scale=torch.zeros(63)), dict(w_scale=torch.zeros(1)), dict(w_scale=torch.zeros(128)[::2]),
                dict(epilogue=K.ACCUMULATE, out=torch.zeros(4, 64, dtype=BF16)), dict(epilogue=silu), dict(epilogue=silu, out=torch.zeros(4, 24), w=eight(48, 32), w_scale=torch.zeros(48)),
                dict(x=eight(4, 0), w=eight(64, 0))):
        with pytest.raises(K.KernelError):
            linear(**bad)
    off = torch.zeros(3, dtype=torch.int32)
    grouped = dict(w=eight(2, 64, 32), w_scale=torch.zeros(2, 64), group_offsets=off)
    for bad in (dict(group_offsets=off.long()), dict(group_offsets=off[:2]), dict(w=eight(64, 32)), dict(w_scale=torch.zeros(128)), dict(w=eight(3, 64, 32)), dict(w=eight(2, 32, 64).transpose(1, 2))):
        with pytest.raises(K.KernelError):
            linear(**{**grouped, **bad})
    assert not calls
    linear(epilogue=silu, out=torch.zeros(4, 32, dtype=BF16))
    linear(x=K.e4m3_rows(4, 30), w=torch.as_strided(eight(5000), (64, 30), (70, 1)))
    linear(x=eight(1, 32).expand(4, 32))
    linear(**grouped)
    linear(**{**grouped, "w": torch.as_strided(eight(20000), (2, 64, 32), (7000, 48, 1))})
    linear(out=torch.zeros(0, 64), x=eight(0, 32), x_scale=torch.zeros(0))
    linear(out=torch.zeros(4, 0), w=eight(0, 32), w_scale=torch.zeros(0))
    linear(w=eight(0, 64, 32), w_scale=torch.zeros(0, 64), group_offsets=off[:1])
    assert [a[6:13] for _, a in calls] == [(4, 64, 32, 32, 32, 32, silu), (4, 64, 30, 32, 70, 64, 0), (4, 64, 32, 0, 32, 64, 0), (4, 64, 32, 32, 32, 64, 0), (4, 64, 32, 32, 48, 64, 0)]
    assert [a[14:16] for _, a in calls] == [(1, 0), (1, 0), (1, 0), (2, 64 * 32), (2, 7000)]


def test_a_refusal_of_the_library_is_raised(monkeypatch):
    """Epilogues that only the library knows to be wrong: its message becomes the error, nothing is launched."""
    monkeypatch.setattr(K, "_not_here", lambda *a, **k: None)
    monkeypatch.setattr(K, "_status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(K, "_stream_on", lambda device: 0)
    for epilogue, out in ((3, torch.zeros(4, 64)), (K.ACCUMULATE | (1 << 8), torch.zeros(4, 64)), (K.plain_act_epilogue(0), torch.zeros(4, 64)), (K.SWIGLU | (9 << 8), torch.zeros(4, 32))):
        with pytest.raises(K.KernelError, match="epilogue"):
            linear(out, epilogue=epilogue)


def test_every_product_has_a_form():
    """Over all sizes, on devices of any number of SMs: pairs for many rows only, else tiles no wider than the rows need, K cut only where every
    block has two stages and all blocks are on the SMs at once."""
    import random
    rng = random.Random(3)
    seen = set()
    for _ in range(20000):
        g, r, N, K_ = (int(2 ** rng.uniform(0, top)) for top in (7, 12, 16, 14))
        sms = rng.choice([1, 2, 74, 148, 148, 148, 160])
        form = K.lib().leb_linear_e4m3_form(g, r, N, K_, sms)
        if form == 0:
            assert r >= 40
            continue
        rows, slices = form & 0xffff, form >> 16
        assert rows in (16, 32, 64, 128) and slices in ((1,) if rows == 128 else (1, 2, 4, 8)) and (rows == 16 or rows < 2 * r)
        blocks = g * -(-r // rows) * -(-N // 128) * slices
        assert slices == 1 or (blocks <= 2 * sms and -(-K_ // 128) >= 2 * slices)
        seen.add((rows, slices > 1))
    assert len(seen) == 7
