"""Windowed prefill with logits of any magnitude: the keys that share a row's
largest logit exactly share its weight, whatever the logit's size and whatever
sizes the row met before; no finite input gives a NaN.

Queries are zero but for one value 2^e and keys hold small whole numbers there,
so logits are exact multiples of 2^e / 8 and for e >= 10 all but the largest
have weights below e^-128.  Tolerance per value: a weight is 2^r with r what the
row's maximum was rounded by, the same for all of them but no power of two,
and is rounded to bf16 (2^-8) for the values and not for its sum; sums are
fp32, the output is bf16: 2^-8 |o| + (2^-8 + 2^-20) mean |v|."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
POWERS = [10, 13, 22, 27, 28, 29, 31, 33, 40, 60, 90, 116]


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from cache_eviction_b200 import capi
    capi.load()


def run(q, k, v, nq, window, first, P, sinks=None):
    """window_prefill of the last nq of n tokens, pages in order."""
    from cache_eviction_b200 import kernels
    n, G = k.shape[:2]
    units = -(-n // P)
    i32 = dict(dtype=torch.int32, device=DEV)
    pools = []
    for x in (k, v):
        pool = torch.full((units * P, G, 64), float("nan"), dtype=torch.bfloat16)
        pool[:n] = x
        pools.append(pool.view(units, P, G, 64).transpose(1, 2).contiguous().to(DEV))
    err = torch.zeros(1, **i32)
    out = kernels.window_prefill(q.to(DEV), *pools, torch.tensor([0, nq], **i32), torch.tensor([0, units], **i32),
                                 torch.arange(units, **i32), torch.tensor([n], **i32), 0.125, P, nq, n, window, first=first,
                                 sinks=None if sinks is None else sinks.to(DEV), err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    return out.double().cpu()


def hold(out, code, sign, v, nq, window, first, heads=slice(None)):
    """Each row against the mean of the values of its visible keys of largest sign * code."""
    n = code.shape[0]
    t = torch.arange(n)
    for i in range(nq):
        p = n - nq + i
        seen = (t <= p) & ((t > p - window) | (t < first)) if window >= 0 else t <= p
        best = seen & (sign * code == (sign * code)[seen].max())
        for g in range(v.shape[1]):
            x = v[best, g].double()
            tol = 2.0 ** -8 * x.mean(0).abs() + (2.0 ** -8 + 2.0 ** -20) * x.abs().mean(0)
            off = ((out[i, 8 * g:8 * g + 8][heads] - x.mean(0)).abs() / tol)
            assert off.max() <= 1, (i, g, off.amax(-1))      # (a NaN fails as well)


@pytest.mark.parametrize("P", [16, 4])
@pytest.mark.parametrize("window,first", [(-1, 0), (150, 20)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("powers", [POWERS[:8], POWERS[4:]])
def test_one_magnitude_a_row(powers, sign, window, first, P):
    gen = torch.Generator().manual_seed(1)
    n, nq, G = 700, 70, 2
    code = torch.randint(3, 20, (n,), generator=gen).float()
    k, v = torch.randn((2, n, G, 64), generator=gen).to(torch.bfloat16)
    k[:, :, 0] = code.view(-1, 1).to(torch.bfloat16)
    q = torch.zeros((nq, 8 * G, 64))
    q[:, :, 0] = sign * 2.0 ** torch.tensor([float(e) for e in powers]).repeat(G)
    hold(run(q.to(torch.bfloat16), k, v, nq, window, first, P), code, sign, v, nq, window, first)


@pytest.mark.parametrize("order", [(-116, -2, 1), (1, -116, -2), (1, 40, 80), (80, 40, 1), (-100, 40, 100), (-2, -116, 1), (40, -40, 41)])
def test_magnitudes_that_change_along_a_row(order):
    """Stretches of keys of very different magnitude, rising and falling from
    tile to tile, among them the lowest that fp32 has: sign(x) 2^|x| times a whole
    number below 32.  (Up, 116 would be no case: 31 * 2^116 * 2^10 / 8 is 2^127.95
    and log2(e) times that is beyond fp32.)"""
    gen = torch.Generator().manual_seed(2)
    n, nq, G = 900, 40, 1
    size = torch.tensor([float(x) for x in order]).repeat_interleave(300)
    code = torch.randint(17, 32, (n,), generator=gen).float() * size.sign() * 2.0 ** size.abs()
    k = torch.zeros((n, G, 64))
    k[:, 0, 0] = code
    v = torch.randn((n, G, 64), generator=gen).to(torch.bfloat16)
    q = torch.zeros((nq, 8, 64))
    q[:, :, 0] = 2.0 ** 10
    hold(run(q.to(torch.bfloat16), k.to(torch.bfloat16), v, nq, -1, 0, 16), code, 1.0, v, nq, -1, 0)


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_sinks_beside_large_logits(sign):
    """A sink of ordinary size takes everything beside large negative logits and
    nothing beside large positive ones."""
    gen = torch.Generator().manual_seed(3)
    n, nq, G = 300, 20, 1
    code = torch.randint(3, 20, (n,), generator=gen).float()
    k, v = torch.randn((2, n, G, 64), generator=gen).to(torch.bfloat16)
    k[:, :, 0] = code.view(-1, 1).to(torch.bfloat16)
    q = torch.zeros((nq, 8, 64))
    q[:, :, 0] = sign * 2.0 ** torch.tensor([10.0, 13.0, 22.0, 28.0, 31.0, 40.0, 90.0, 116.0])
    out = run(q.to(torch.bfloat16), k, v, nq, -1, 0, 16, sinks=torch.randn(8, generator=gen))
    if sign > 0:
        hold(out, code, sign, v, nq, -1, 0)
    else:
        assert (out == 0).all()
