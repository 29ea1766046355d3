"""Page lists that name no page where a row reads: no address is formed from that, whatever kernel the step goes to."""
import types

import pytest
import torch

import harness as H  # noqa: F401  (path setup)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("new", [1, 3, 40, 200])
@pytest.mark.parametrize("dtype,nh,nkv,hd,page,kw", [
    (BF16, 8, 2, 64, 64, {}), (BF16, 8, 2, 64, 64, {"wide": True}), (BF16, 8, 2, 128, 64, {}), (BF16, 4, 2, 32, 32, {}), (BF16, 2, 2, 96, 32, {"wide": True}),
    (BF16, 4, 2, 80, 64, {}), (F32, 4, 2, 64, 64, {}), (F32, 3, 1, 48, 32, {})])
@pytest.mark.parametrize("window,chunk,first", [(90, 0, 70), (0, 128, 3), (64, 100, 1)])
def test_rows_that_read_pages_given_back(new, dtype, nh, nkv, hd, page, kw, window, chunk, first):
    """What is read there is not said (another page, or zeros); results are finite where every page's numbers are, and the other
    sequence's are what they were."""
    from lastengine_b200.ops import kernels as K
    word = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    B, held = 2, 300
    width = -(-(held + new) // page)
    g = torch.Generator(device=DEV).manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)
    q, k, v = rand(B * new, nh * hd), rand(B * width, nkv, page, hd), rand(B * width, nkv, hd, page)
    whole = torch.arange(B * width, dtype=torch.int32, device=DEV).view(B, width)
    batch = types.SimpleNamespace(n_rows=B * new, n_seqs=B, max_qlen=new, max_kvlen=held + new, row_seq=word([0] * new + [1] * new),
                                  row_pos=word([held + i for i in range(new)] * 2), seq_slot=word([0, 1]), seq_pos0=word([held] * 2),
                                  seq_qstart=word([0, new]), seq_qlen=word([new] * 2))

    def run(table):
        out = torch.full((B * new, nh * hd), float("nan"), dtype=dtype, device=DEV)
        K.attention(out, q, k, v, table, batch, nh, nkv, hd, page, window, hd ** -0.5, chunk=chunk, first=first, **kw)
        K.check_device_status()
        return out

    want = run(whole)
    for lost in ([0], [width - 2], list(range(width - 1)), list(range(width))):
        table = whole.clone()
        table[0, lost] = -1
        got = run(table)
        assert bool(torch.isfinite(got).all())
        assert torch.equal(got[new:], want[new:])
