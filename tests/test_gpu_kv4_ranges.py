"""4-bit decode attention where the ranges of fp32 and fp16 could end: value
rows of one value, scales far apart, rows that nobody looks at, logits of any
magnitude, query rows near the largest bf16, and long rows in one block.

Everything is held to attention over the same pages in 64 bits.  Tolerances,
from the arithmetic, as in test_gpu_kv4.py: a logit is off by at most
d = 80 * 2^-24 * scale * (s sum |q| c + |m| sum |q|), a p by the relative
e = 2 d + 16 * 2^-24 * (1 + |logit range|); p s is rounded to fp16 (2^-11
relative; below fp16's normal range 2^-25, where the largest p s of the row is
at least 2^7, so 2^-32 of that one); the output to bf16 (2^-8):

    |error| <= 2^-8 |o| + (2^-11 + e) sum p s c + (e + A 2^-24) sum p |m|
               + 2^-32 n 15 max(p s)

with A the additions that a term of sum p m goes through (at most n / 8 in a
lane and 64 after that).
"""
import math

import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 0.125


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from cache_eviction_b200 import capi
    capi.load()


def slices(x, is_key):
    """Tokens x [n, G, 64] bf16 as pages [ceil(n / 16), G, 576] (the rest of the last page zeros)."""
    n, G = x.shape[:2]
    full = torch.zeros((-(-n // 16) * 16, G, 64), dtype=torch.bfloat16)
    full[:n] = x
    return ref.pack(*ref.quantise(full.view(-1, 16, G, 64).transpose(1, 2)), is_key)


def one_row(q, kp, vp, n, sinks=None):
    """The operator over one row of n tokens in pages 0, 1, ... -> out [H, 64], lse [H] (64 bits, host)."""
    from cache_eviction_b200 import kernels
    units, G = kp.shape[:2]
    i32 = dict(dtype=torch.int32, device=DEV)
    lse, err = torch.empty((1, 8 * G), device=DEV), torch.zeros(1, **i32)
    out = kernels.kv4_decode_attn_score(q[None].to(DEV), kp.to(DEV), vp.to(DEV), torch.tensor([0, units], **i32),
                                        torch.arange(units, **i32), torch.tensor([n], **i32), SCALE,
                                        sinks=None if sinks is None else sinks.to(DEV), lse=lse, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    return out[0].double().cpu(), lse[0].double().cpu()


def hold(q, kp, vp, n):
    """one_row against the 64-bit form, every head."""
    out, lse = one_row(q, kp, vp, n)
    for g in range(kp.shape[1]):
        (kc, ks, km), (vc, vs, vm) = ((x.reshape(-1, x.shape[-1])[:n] for x in ref.unpack(t[:, g], key))
                                      for t, key in ((kp, True), (vp, False)))
        hs = slice(8 * g, 8 * g + 8)
        qq = q[hs].double()
        p, o, l = ref.attend(qq[None], km + kc * ks, vm + vc * vs, torch.ones(1, n, dtype=torch.bool), None, SCALE)
        p, o, l = p[0], o[0], l[0]
        d = 80 * 2.0 ** -24 * SCALE * (qq.abs() @ kc.T * ks.T + qq.abs().sum(-1, keepdim=True) * km.abs().T).amax(-1)
        logits = qq @ (km + kc * ks).T * SCALE
        e = (2 * d + 16 * 2.0 ** -24 * (1 + (logits - l[:, None]).abs().amax(-1)))[:, None]
        assert (e < 0.25).all()      # a tolerance that tells something
        tol = (2.0 ** -8 * o.abs() + (2.0 ** -11 + e) * (p @ (vc * vs)) + (e + (n / 8 + 64) * 2.0 ** -24) * (p @ vm.abs())
               + 2.0 ** -32 * n * 15 * (p * vs.T).amax(-1, keepdim=True) + 1e-37)
        assert ((out[hs] - o).abs() <= tol).all(), (g, float(((out[hs] - o).abs() / tol).nan_to_num(1e9).max()))
        assert ((lse[hs] - l).abs() <= e[:, 0] + 2.0 ** -22 * (1 + l.abs())).all()


def draws(n, G, seed):
    gen = torch.Generator().manual_seed(seed)
    k = (torch.randn((n, G, 64), generator=gen) + 0.5 * torch.randn((1, G, 64), generator=gen)).to(torch.bfloat16)
    v = torch.randn((n, G, 64), generator=gen)
    return (torch.randn((8 * G, 64), generator=gen) * 1.5).to(torch.bfloat16), k, v


# ------------------------------------------------------------ value rows of one value
@pytest.mark.parametrize("G", [1, 8])
@pytest.mark.parametrize("n", [1, 700, 70003])
@pytest.mark.parametrize("value", [0.0, 1.0, 3e3, 1e7, -1e7, 1e30, -3e38])
def test_value_rows_of_one_value(value, n, G):
    """Every value row is constant (scale 0): the output is that value.  Its
    terms p m and the sum of p pass through at most n / 8 + 64 additions each."""
    q, k, _ = draws(n, G, n + G)
    v = torch.full((n, G, 64), value, dtype=torch.bfloat16)
    out, _ = one_row(q, slices(k, True), slices(v, False), n)
    want = v.double()[0, 0, 0]
    tol = (2.0 ** -8 + 2 * (n / 8 + 64) * 2.0 ** -24) * want.abs()
    assert ((out - want).abs() <= tol).all(), out


@pytest.mark.parametrize("G,n", [(1, 700), (8, 700), (2, 20011)])
@pytest.mark.parametrize("value", [0.0, 1e4, -1e7, 1e30])
@pytest.mark.parametrize("spread", [1.0, 2.0 ** 60, 2.0 ** 110])
def test_constant_rows_before_and_after_others(value, spread, G, n):
    """What came before counts, however far the scales that follow are from its."""
    q, k, v = draws(n, G, 3)
    kp = slices(k, True)
    for some in (slice(0, n // 2 + 3), slice(n // 2 + 3, n)):
        x = v * spread
        x[some] = value
        hold(q, kp, slices(x.to(torch.bfloat16), False), n)


@pytest.mark.parametrize("G", [1, 8])
@pytest.mark.parametrize("power", [20, 40, 100])
@pytest.mark.parametrize("at", [0, 350, 699])
def test_a_large_value_row_that_heads_do_not_see(at, power, G):
    """One value row is 2^power times the others; half of the heads give it a
    weight near 0 and keep the others' contributions, half see little else."""
    n = 700
    q, k, v = draws(n, G, 5)
    sign = torch.tensor([1.0, -1.0]).repeat(4 * G)
    q[:, :8] = (4 * sign[:, None]).to(torch.bfloat16)
    k[:, :, :8] = 0
    k[at] = 0
    k[at, :, :8] = -40.0                       # logits of 8 * 4 * 40 / 8 = 160, down or up
    v[at] *= 2.0 ** power
    hold(q, slices(k, True), slices(v.to(torch.bfloat16), False), n)


@pytest.mark.parametrize("G,n", [(1, 700), (8, 2011)])
@pytest.mark.parametrize("zeros", [0, 300, 690, 10 ** 6])
@pytest.mark.parametrize("rise", [-400.0, 40.0, 400.0])
def test_logits_that_rise_or_fall_along_a_row(rise, zeros, G, n):
    """Logits that change by `rise` over the row, its first value rows zeros:
    weights of rows that add nothing grow as well."""
    q, k, v = draws(n, G, 6)
    q[:, :8] = 4.0
    k[:, :, :8] = (rise / 4.0 * (torch.arange(n) / n - 0.5)).view(-1, 1, 1)     # logit 4 * 8 / 8 of it
    v[:zeros] = 0.0
    hold(q, slices(k, True), slices(v.to(torch.bfloat16), False), n)


@pytest.mark.parametrize("G", [1, 8])
def test_long_rows_in_one_block(G):
    """More rows than blocks, 8K to 32K tokens each over the same pages, so that
    a block adds up whole rows.  Keys are 0: every p is 1 and p s exact in fp16,
    and what is left is the sums of p s c and p m, whose terms cancel (the values
    have mean 0).  Of a sum of positive terms the tensor cores lose at most
    2^-19 over the 32 tokens that they add up at a time (two products of 16,
    whose terms they cut to 24 bits at the largest one's), every addition in
    fp32 2^-24: n / 32 of them and 64 after, n / 8 and 64 for p m."""
    from cache_eviction_b200 import kernels
    B, T = 320, 32768
    gen = torch.Generator().manual_seed(30 + G)
    vp = slices(torch.randn((T, G, 64), generator=gen).to(torch.bfloat16), False)
    kp = torch.zeros_like(vp)
    lens = torch.tensor([T - (i * 7919) % 24577 for i in range(B)])
    counts = -(-lens // 16)
    i32 = dict(dtype=torch.int32, device=DEV)
    indptr = torch.cat((torch.zeros(1, dtype=torch.int64), counts.cumsum(0))).to(**i32)
    indices = torch.cat([torch.arange(c) for c in counts]).to(**i32)
    q = torch.randn((B, 8 * G, 64), generator=gen).to(torch.bfloat16).to(DEV)
    out = kernels.kv4_decode_attn_score(q, kp.to(DEV), vp.to(DEV), indptr, indices, lens.to(**i32), SCALE).double().cpu()
    n = lens.double().view(-1, 1, 1)
    for g in range(G):
        c, s, m = (x.reshape(T, -1) for x in ref.unpack(vp[:, g], False))
        mean, above, low = (x.cumsum(0)[lens - 1][:, None] / n for x in (m + c * s, c * s, m.abs()))
        tol = (2.0 ** -8 * mean.abs() + (2.0 ** -19 + (n / 32 + 64) * 2.0 ** -24) * above + (n / 8 + 64) * 2.0 ** -24 * low)
        off = ((out[:, 8 * g:8 * g + 8] - mean).abs() / tol).view(B, 8, 4, 2, 8).amax((0, 1, 2, 4))
        assert (off <= 1).all(), (g, off)      # dims 0 .. 7 and 8 .. 15 of every 16


@pytest.mark.parametrize("G,n", [(1, 700), (8, 2011)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_logits_of_any_magnitude(sign, G, n):
    """Logits (1 + c) 2^e / 8 with c the first code of a key, e from 6 to 116 by
    head, up or down: three keys share the largest one exactly, the next is
    2^e / 8 below, so the output is the mean of three value rows, whose scales
    are 2^-20, 1 and 2^20, within the fp16 rounding of each and the output's."""
    gen = torch.Generator().manual_seed(9)
    units = -(-n // 16)
    best = [5, n // 2, n - 1]
    code = torch.randint(0, 16, (units * 16, G, 64), generator=gen)
    first = torch.randint(0, 15, (units * 16, G), generator=gen)
    first[best] = 15
    code[..., 0] = first if sign > 0 else 15 - first
    one = torch.ones((units, G, 16), dtype=torch.bfloat16)
    paged = lambda x: x.view(units, 16, G, -1).transpose(1, 2)
    kp = ref.pack(paged(code).to(torch.uint8), one, one, True)
    v = torch.randn((n, G, 64), generator=gen)
    for at, power in zip(best, (-20, 0, 20)):
        v[at] *= 2.0 ** power
    vp = slices(v.to(torch.bfloat16), False)
    power = torch.tensor([6.0, 10.0, 22.0, 25.0, 28.0, 34.0, 60.0, 116.0]).repeat(G)
    q = torch.zeros((8 * G, 64))
    q[:, 0] = sign * 2.0 ** power
    out, lse = one_row(q.to(torch.bfloat16), kp, vp, n)
    top = sign * 2.0 ** power.double() / 8 * (16 if sign > 0 else 1) + math.log(3)
    alone = torch.arange(8 * G) % 8 > 0            # 2^6 / 8 = 8 apart, e^-8: the first head sees others
    assert ((lse - top).abs() <= 2.0 ** -21 * (1 + top.abs()))[alone].all()
    for g in range(G):
        c, s, m = (x.reshape(-1, x.shape[-1])[best] for x in ref.unpack(vp[:, g], False))
        mean = (m + c * s).mean(0)
        tol = 2.0 ** -8 * mean.abs() + 2.0 ** -11 * (c * s).mean(0) + 2.0 ** -20 * (c * s + m.abs()).mean(0)
        got = out[8 * g + 1:8 * g + 8]
        assert ((got - mean).abs() <= tol).all(), ((got - mean).abs() / tol).amax(-1)
    hold(q.to(torch.bfloat16)[::8].repeat_interleave(8, 0), kp, vp, n)


@pytest.mark.parametrize("G,n", [(1, 700), (8, 2011)])
def test_value_scales_near_the_end_of_the_range(G, n):
    """V scales beyond 2^68 and up to 2^122, where the weights of keys that count
    for the normaliser would leave fp32 if the sum shared the values' lift."""
    q, k, v = draws(n, G, 10)
    for power in (70, 100, 120):
        x = (v * 2.0 ** power).to(torch.bfloat16)
        hold(q, slices(k, True), slices(x, False), n)


@pytest.mark.parametrize("G", [1, 8])
@pytest.mark.parametrize("power", [110, 117, 118, 121, 125])
def test_query_rows_near_the_largest_bf16(power, G):
    """Query rows of 2^power times ordinary values against keys of 2^-power."""
    q, k, v = draws(700, G, 11)
    q = (q.float() / 4 * 2.0 ** power).to(torch.bfloat16)
    hold(q, slices((4 * k.float() * 2.0 ** -power).to(torch.bfloat16), True), slices(v.to(torch.bfloat16), False), 700)


@pytest.mark.parametrize("G,n", [(1, 700), (8, 2011)])
@pytest.mark.parametrize("power", [-6, -12, -40])
@pytest.mark.parametrize("logit", [3.0, 10.0, 40.0])
def test_a_first_key_of_most_weight_and_small_values(logit, power, G, n):
    """The first key takes most of the weight, or nearly all of it, and its
    values are 2^power of the others'."""
    q, k, v = draws(n, G, 12)
    q[:, :8] = 4.0
    k[:, :, :8] = 0.0
    k[0] = 0.0
    k[0, :, :8] = logit / 4.0
    v[0] *= 2.0 ** power
    hold(q, slices(k, True), slices(v.to(torch.bfloat16), False), n)
