"""Products in 8 bits of operands that TMA does not take, with so many rows that the blocks of a later expert would begin beyond 2^31."""
import pytest
import torch

import harness as H  # noqa: F401  (path setup)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn


def test_experts_behind_a_billion_rows():
    """One number a row, so that a result is one product of whole numbers.  Every expert has blocks for all M rows, counted from its own first
    row: the last expert's go up to 2 M - 1003 = 2.4e9."""
    from lastengine_b200.ops import kernels as K
    M = 1_200_000_000
    ends = [M - 1000, M - 400, M - 3]
    off = torch.tensor([0, *ends], dtype=torch.int32, device=DEV)
    x = torch.empty(M, 1, dtype=E4M3, device=DEV)
    numbers = torch.arange(-8, 9, device=DEV).float().to(E4M3).view(torch.uint8)
    piece = numbers.repeat(1_000_003)
    bytes_ = x.view(torch.uint8).view(-1)
    for lo in range(0, M, piece.numel()):
        n = min(piece.numel(), M - lo)
        bytes_[lo:lo + n] = piece[:n]
    w = torch.tensor([3.0, -5.0, 7.0], device=DEV).to(E4M3).view(3, 1, 1)
    out = torch.full((M, 1), 0.5, dtype=torch.bfloat16, device=DEV)
    K.linear_e4m3(out, x, torch.ones(M, device=DEV), w, torch.ones(3, 1, device=DEV), group_offsets=off)
    lo = 0
    for e, hi in enumerate(ends):
        for a in range(lo, hi, 1 << 27):
            b = min(hi, a + (1 << 27))
            assert torch.equal(out[a:b, 0].float(), x[a:b, 0].float() * float(w[e]))
        lo = hi
    assert bool((out[lo:] == 0.5).all())
    K.check_device_status()
