"""Which kernel a step with first positions goes to: one that takes the step's sizes, addresses and row counts, whatever they are."""
import itertools
import types

import pytest
import torch

import harness as H  # noqa: F401  (path setup)
from lastengine_b200.ops import kernels as K

BF16, F32 = torch.bfloat16, torch.float32


class Place:
    """Where a tensor of the step lies, without its memory."""

    def __init__(self, dtype, shape, at=0):
        self.dtype, self.shape, self.at = dtype, shape, at

    def data_ptr(self):
        return 1 << 20 | self.at

    def stride(self, d):
        return self.shape[1] if d == 0 else 1

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n


def form_of(dtype, nh, nkv, hd, vd, page, M, B, longest, rows_at=0, pools_at=0, wide=False, keys=40, n_pages=10):
    batch = types.SimpleNamespace(n_rows=M, n_seqs=B, max_qlen=longest)
    out, q = Place(dtype, (M, nh * vd), rows_at), Place(dtype, (M, nh * hd), rows_at)
    k, v = Place(dtype, (n_pages, nkv, page, hd), pools_at), Place(dtype, (n_pages, nkv, vd, page), pools_at)
    return K._stream_form(out, batch, nh, nkv, hd, vd, page, wide, q, k, v, keys)


def takes(form, dtype, nh, nkv, hd, vd, page, M, B, longest, rows_at, pools_at, wide):
    """What the kernels' loads and grids ask for."""
    L, G = K.lib(), nh // nkv
    mma = dtype is BF16 and hd == vd and hd in (32, 64, 96, 128) and page % 32 == 0 and rows_at % 16 == 0 and pools_at % 16 == 0
    if form is None:                                   # mma.sync over all rows, or the tcgen05 kernel of weights of two terms
        return mma and G <= 64 and B <= 65535
    if form is K._attention_stream_decode:
        return mma and G <= 16 and longest == 1 and M == B
    if form is K._attention_stream_tc:
        return (dtype is BF16 and rows_at % 16 == 0 and pools_at % 16 == 0 and not wide and longest > 1 and B <= 65535 and -(-longest // (128 // G // 8 * 8)) <= 65535
                and L.leb_attention_stream_tc_supported(nh, nkv, hd, vd, page))
    if form is K._attention_stream_rows:
        return pools_at % 16 == 0 and B <= 65535 and G <= 64 and -(-longest // (64 // G)) <= 65535 and max(hd, vd) <= 256 and page % 32 == 0
    if form is K._attention_stream_any:
        return pools_at % 16 == 0 and M <= 65535 and max(hd, vd) <= 256 and page % 32 == 0
    return form is K._attention_stream_general


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nh,nkv,hd,vd,page", [(1, 1, 32, 32, 32), (1, 1, 32, 32, 64), (2, 1, 64, 64, 64), (32, 8, 64, 64, 64), (16, 1, 128, 128, 64), (34, 2, 64, 64, 64),
                                               (40, 1, 96, 96, 32), (64, 1, 32, 32, 64), (4, 2, 72, 40, 64), (5, 5, 33, 33, 32), (3, 1, 192, 192, 64), (130, 1, 64, 64, 64)])
def test_every_step_goes_to_a_kernel_that_takes_it(dtype, nh, nkv, hd, vd, page):
    steps = [(1, 1, 1), (7, 7, 1), (5, 7, 1), (65535, 65535, 1), (30, 3, 20), (65535, 1, 65535), (65536, 1, 65536), (70000, 1, 70000), (70000, 60000, 9), (70000, 69000, 9),
             (600000, 1, 600000), (2200000, 2, 2100000), (40, 39, 2)]
    for (M, B, longest), rows_at, pools_at, wide in itertools.product(steps, (0, 2, 8), (0, 4), (False, True)):
        if B > 65535:      # more sequences than any kernel takes: what is chosen says so
            continue
        args = (dtype, nh, nkv, hd, vd, page, M, B, longest, rows_at, pools_at, wide)
        try:
            form = form_of(*args)
        except K.KernelError:
            assert pools_at and dtype is BF16 and hd == vd and hd in (32, 64, 96, 128)
            continue
        assert takes(form, *args), (form and form.__name__, args)


def test_many_rows_that_begin_anywhere_do_not_go_to_the_kernels_of_16_byte_loads():
    assert form_of(BF16, 1, 1, 32, 32, 32, 70000, 1, 70000) is None
    assert form_of(BF16, 1, 1, 32, 32, 32, 70000, 1, 70000, rows_at=2) is K._attention_stream_rows
    assert form_of(BF16, 1, 1, 64, 64, 64, 70000, 1, 70000, rows_at=8, keys=20) is K._attention_stream_rows
    assert form_of(F32, 1, 1, 32, 32, 32, 70000, 1, 70000, pools_at=4) is K._attention_stream_general
    assert form_of(F32, 64, 1, 32, 32, 32, 70000, 1, 70000) is K._attention_stream_general


@pytest.mark.parametrize("source", ["attention.cu", "attention_decode.cu", "attention_prefill.cu", "attention_prefill_tc.cu", "attention_stream_any.cu",
                                    "attention_stream_rows.cu", "attention_stream_tc.cu", "stream_tables.cu"])
def test_shared_memory_is_allowed_on_every_device_that_launches_a_kernel(source):
    """The limit belongs to a device's copy of a kernel: it is raised by leb_allow_smem, which keeps count of devices, and behind no flag of the
    whole process."""
    import os
    from lastengine_b200.ops import build
    with open(os.path.join(build.CSRC, source)) as f:
        text = f.read()
    assert "cudaFuncSetAttribute" not in text
    assert "leb_allow_smem" in text or "extern __shared__" not in text


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nh,nkv,hd,vd", [(8, 2, 64, 64), (32, 8, 64, 64), (32, 8, 64, 48), (16, 1, 128, 128), (34, 2, 64, 64), (4, 2, 80, 80), (4, 4, 192, 192), (6, 6, 96, 32)])
@pytest.mark.parametrize("B", [1, 8, 64, 300])
@pytest.mark.parametrize("window,chunk", [(4096, 0), (0, 2048)])
def test_splits_through_scratch_are_asked_for_only_where_they_are_read(dtype, nh, nkv, hd, vd, B, window, chunk):
    batch = types.SimpleNamespace(n_rows=B, n_seqs=B, max_qlen=1, max_kvlen=9000)
    n = K.attention_splits(batch, nkv, nh // nkv, sm_count=148, hd=hd, window=window, chunk=chunk, general=dtype is F32 or vd != hd, first=4)
    form = form_of(dtype, nh, nkv, hd, vd, 64, B, B, 1, keys=4100)
    assert n == 1 or form is K._attention_stream_decode
    if form is K._attention_stream_decode and B * nkv >= 2 * 148:
        assert n == (4 if window else 2)
