"""kv4_write on rows whose span max - min lies beyond fp32's end: the codes are
those of the format in 64 bits, c = clamp(rint((x - m) / s), 0, 15)."""
import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("high", [1.8e38, 3.0e38, 3.38e38])
def test_codes_of_rows_wider_than_fp32(high):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(1)
    T = 160
    x = ((2 * torch.rand((T, 1, 64), generator=gen, dtype=torch.float64) - 1) * high).to(torch.bfloat16)
    x[:, 0, 3], x[:, 0, 40] = -high, high
    pool = torch.zeros((2, T // 16, 1, 576), dtype=torch.uint8, device=DEV)
    kernels.kv4_write(x.to(DEV), x.to(DEV), pool[0], pool[1], torch.arange(T, device=DEV))
    d = x.double()[:, 0]
    low, top = d.amin(-1, keepdim=True), d.amax(-1, keepdim=True)
    assert ((top - low) > 3.41e38).all()
    scale = ((top / 2 - low / 2) * (2 / 15)).to(torch.bfloat16).double()
    quotient = (d - low) / scale
    clear = (quotient - quotient.floor() - 0.5).abs() > 2.0 ** -20     # ties and what rounds to one in fp32
    want = torch.round(quotient).clamp(0, 15)
    assert clear.float().mean() > 0.95
    for kv, key in ((0, True), (1, False)):
        c, s, m = (t.view(T, -1) for t in ref.unpack(pool[kv].cpu()[:, 0], key))
        assert torch.equal(s, scale) and torch.equal(m, low)
        assert torch.equal(c[clear], want[clear])
