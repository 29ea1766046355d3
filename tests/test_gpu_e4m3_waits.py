"""8-bit products whose bounded waits give up: the blocks leave in order (their copies have landed, their products are done, tensor memory is
free), the status word says so, and the context goes on.  The kernels are built once more with waits that give up at random moments."""
import ctypes
import os
import subprocess

import pytest
import torch

import harness as H  # noqa: F401  (path setup)
from test_gpu_stream_waits import STUB

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def impatient(tmp_path_factory):
    """leb_linear_e4m3 with waits of which one in some two thousand is given up at once, by the clock."""
    from lastengine_b200.ops import build
    d = tmp_path_factory.mktemp("impatient")
    (d / "stub.cu").write_text(STUB)
    so = str(d / "impatient.so")
    files = [os.path.join(build.CSRC, f"gemm_e4m3{n}.cu") for n in ("", "_few", "_pairs", "_any")]
    subprocess.run([build._find_nvcc(), *build.NVCC_FLAGS, "-I", build.CSRC, "-DTC_SPIN_LIMIT=(((unsigned)clock64() >> 4) % 1999u ? 1u << 22 : 0u)", "-DE8_PATIENT=0",
                    "-shared", "-o", so, *files, str(d / "stub.cu")], check=True, timeout=600)
    lib = ctypes.CDLL(so)
    lib.leb_linear_e4m3.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
    lib.leb_last_error.restype = ctypes.c_char_p
    return lib


# (rows, columns, K, rows of every expert or None): the weights-first kernel walking tiles, with a cluster a tile, grouped; pairs, dense and grouped
CASES = {"tiles": (20, 60000, 256, None), "clusters": (40, 512, 4096, None), "experts": (200, 1000, 512, [50, 0, 90, 60]),
         "pairs": (1500, 4000, 1024, None), "pairs, experts": (2000, 1500, 512, [700, 0, 900, 400])}


@pytest.mark.parametrize("name", CASES)
def test_a_wait_that_gives_up_leaves_in_order(impatient, name):
    from lastengine_b200.ops import kernels as K
    M, N, K_, counts = CASES[name]
    E = len(counts) if counts else 1
    g = torch.Generator(device=DEV).manual_seed(1)
    whole = lambda *s: torch.randint(-8, 9, s, generator=g, device=DEV).float().to(E4M3)  # noqa: E731
    x, w = whole(M, K_), whole(E * N, K_)
    sx, sw = torch.ones(M, device=DEV), torch.ones(E * N, device=DEV)
    off = torch.tensor([sum(counts[:e]) for e in range(E + 1)], dtype=torch.int32, device=DEV) if counts else None
    out, status = torch.empty(M, N, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)

    def run(L):
        packed = K._PACK_LINEAR(out.data_ptr(), K.F32, x.data_ptr(), sx.data_ptr(), w.data_ptr(), sw.data_ptr(), M, N, K_, K_, K_, N, K.STORE,
                                off.data_ptr() if counts else 0, E, N * K_, status.data_ptr())
        assert L.leb_linear_e4m3(packed, torch.cuda.current_stream().cuda_stream) == 0, L.leb_last_error()
        code = int(status)
        status.zero_()
        return out.clone(), code

    want, code = run(K.lib())
    assert code == 0
    gave_up = went_through = 0
    for _ in range(60):
        got, code = run(impatient)
        if code:
            assert code in (51, 52, 53, 54, 55, 61, 62, 63, 64)
            gave_up += 1
        else:
            assert torch.equal(got, want)
            went_through += 1
        got, code = run(K.lib())
        assert code == 0 and torch.equal(got, want)
    assert gave_up >= 3, (gave_up, went_through)
