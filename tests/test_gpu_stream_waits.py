"""Prompt attention with first positions whose bounded waits give up: the block leaves in order (its copies have landed, its products are done, its
tensor memory is free), the status word says so, and the context goes on.  The kernel is built once more with waits that give up at random moments."""
import ctypes
import os
import subprocess
import types

import pytest
import torch

import harness as H  # noqa: F401  (path setup)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16

STUB = r"""
#include <stdarg.h>
#include <string.h>
#include "common.cuh"
long long g_leb_launches = 0;
int g_leb_pdl = 1;
thread_local int g_leb_gate_act = 0;
static char message[512];
int leb_fail(const char* fmt, ...) { va_list a; va_start(a, fmt); vsnprintf(message, sizeof message, fmt, a); va_end(a); return 1; }
LEB_API const char* leb_last_error() { return message; }
extern "C" int leb_sm_count() { int n = 0; cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, 0); return n; }
"""


@pytest.fixture(scope="module")
def impatient(tmp_path_factory):
    """leb_attention_stream_tc with waits of which one in some hundreds is given up at once, by the clock."""
    from lastengine_b200.ops import build, kernels
    d = tmp_path_factory.mktemp("impatient")
    (d / "stub.cu").write_text(STUB)
    so = str(d / "impatient.so")
    subprocess.run([build._find_nvcc(), *build.NVCC_FLAGS, "-I", build.CSRC, "-DTC_SPIN_LIMIT=(((unsigned)clock64() >> 4) % 599u ? 1u << 22 : 0u)", "-shared", "-o", so,
                    os.path.join(build.CSRC, "attention_stream_tc.cu"), str(d / "stub.cu")], check=True, timeout=300)
    lib = ctypes.CDLL(so)
    lib.leb_attention_stream_tc.argtypes = kernels.lib().leb_attention_stream_tc.argtypes
    lib.leb_last_error.restype = ctypes.c_char_p
    return lib


@pytest.mark.parametrize("nh,nkv,hd,vd", [(8, 2, 64, 64), (4, 2, 128, 128), (4, 2, 72, 40)])
def test_a_wait_that_gives_up_leaves_in_order(impatient, nh, nkv, hd, vd):
    from lastengine_b200.ops import kernels as K
    word = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    page, window, first = 64, 700, 70
    gave_up = went_through = 0
    for held, new in ((500, 20), (900, 100), (0, 300)):
        n = -(-(held + new) // page)
        rand = lambda *s: torch.randn(s, generator=g, device=DEV).to(BF16)
        q, k, v = rand(new, nh * hd), rand(n, nkv, page, hd), rand(n, nkv, vd, page)
        table, slot, pos0, start, qlen = torch.arange(n, dtype=torch.int32, device=DEV)[None], word([0]), word([held]), word([0]), word([new])
        out, status = torch.empty(new, nh * vd, dtype=BF16, device=DEV), word([0])

        def run(L, splits):
            rc = L.leb_attention_stream_tc(out.data_ptr(), q.data_ptr(), q.stride(0), new, k.data_ptr(), v.data_ptr(), n, table.data_ptr(), n, slot.data_ptr(),
                                           pos0.data_ptr(), start.data_ptr(), qlen.data_ptr(), None, 0, 0, 1, nh, nkv, hd, vd, page, window, 0, first, hd ** -0.5,
                                           None, None, new, held + new, splits, status.data_ptr(), torch.cuda.current_stream().cuda_stream)
            assert rc == 0, L.leb_last_error()
            return out.clone(), int(status)

        for splits in (1, 3):
            want, code = run(K.lib(), splits)
            assert code == 0
            for _ in range(60):
                got, code = run(impatient, splits)
                status.zero_()
                if code:
                    assert 31 <= code <= 42
                    gave_up += 1
                else:
                    assert torch.equal(got, want)
                    went_through += 1
            got, code = run(K.lib(), splits)
            assert code == 0 and torch.equal(got, want)
    assert gave_up >= 10 and went_through >= 10, (gave_up, went_through)
