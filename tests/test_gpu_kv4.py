"""The 4-bit KV cache on the GPU: ce_kv4_write and ce_kv4_read bit for bit
against the page format stated in plain torch, ce_kv4_decode_attn_score
against attention over the same pages in 64 bits.

Tolerances of the attention (per value, from the arithmetic):
  * a logit is s (q . c) + m sum q in fp32: 64 products and sums and a handful
    of further roundings, each at most 2^-24 of the terms' magnitude, so it is
    off by at most d = 80 * 2^-24 * scale * (s sum |q| c + |m| sum |q|); every p
    is off by at most the relative e = 2 d (its own and the normaliser's) plus
    16 * 2^-24 * (1 + |logit range|) for the exponentials and sums;
  * p s is rounded to fp16 (2^-11 relative, 2^-25 * 2^-14 of the largest
    below fp16's normal range) before it meets the codes, the output to bf16
    (2^-8): |error| <= 2^-8 |o| + (2^-11 + e) sum p s c + e sum p |m| + tiny;
  * scores and normalisers are fp32 sums of p: relative e, plus 2^-23 times
    the log2 masses' magnitude for what passes through a logarithm.
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


def same_bits(a, b):
    """Equal values, NaN where NaN (bf16)."""
    a, b = a.float(), b.float()
    return bool(torch.equal(a.isnan(), b.isnan()) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)))


def special_rows(T, G, gen):
    """Rows of ordinary values, and among them the ones that go wrong first."""
    x = torch.randn((T, G, 64), generator=gen) * torch.exp(torch.randn((T, G, 1), generator=gen))
    x[0 % T] = 0.0
    x[1 % T] = -3.25                                  # constant: scale 0
    x[2 % T] *= 1e30
    x[3 % T] = x[3 % T].sign() * 3.3e38               # max - min beyond fp32
    x[4 % T] *= 1e-39                                 # subnormal
    x[5 % T, :, :] = torch.arange(64) / 2.0 - 8.0     # many ties
    x[6 % T, :, 63] = 1e4                             # one outlier
    x = x.to(torch.bfloat16)
    if T > 9:
        x[7, :, 5] = float("nan")
        x[8, :, 0] = float("inf")
        x[9, :, 63] = float("-inf")
    return x


@pytest.mark.parametrize("T,G", [(1, 8), (3, 1), (16, 2), (17, 8), (64, 8), (257, 4), (1000, 3)])
@pytest.mark.parametrize("run", ["scattered", "run", "offset run", "two runs", "runs with padding"])
def test_write_then_read_is_the_format(T, G, run):
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(T * 10 + G)
    units = -(-T // 16) + 5
    k, v = special_rows(T, G, gen), special_rows(T, G, gen).flip(2)
    pools = [ref.random_pool(units, G, key, gen) for key in (True, False)]
    order = torch.randperm(units, generator=gen)
    slots = (order[:, None] * 16 + torch.arange(16)).view(-1)      # consecutive positions of scattered units
    if run == "scattered":
        loc = torch.randperm(units * 16, generator=gen)[:T]
    elif run == "two runs":
        loc = torch.cat((slots[7:7 + T // 2], slots[units * 16 - (T - T // 2):]))
    else:
        loc = slots[(0 if run == "run" else 21):][:T].clone()
    written = torch.ones(T, dtype=torch.bool)
    if run == "runs with padding":
        written[torch.randperm(T, generator=gen)[:T // 5]] = False
        loc[~written] = -1
    dk, dv = pools[0].to(DEV), pools[1].to(DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    kernels.kv4_write(k.to(DEV), v.to(DEV), dk, dv, loc.to(DEV), err=err)
    k, v, loc = k[written], v[written], loc[written]
    want = []
    for pool, x, key in ((pools[0], k, True), (pools[1], v, False)):
        c, s, m = ref.unpack(pool, key)
        c, s, m = c.to(torch.uint8), s[..., 0].to(torch.bfloat16), m[..., 0].to(torch.bfloat16)
        nc, ns, nm = ref.quantise(x)
        c[loc // 16, :, loc % 16], s[loc // 16, :, loc % 16], m[loc // 16, :, loc % 16] = nc, ns, nm
        want.append(ref.pack(c, s, m, key))
    # the slices' bytes: codes, scales and minima where the format has them,
    # every slot that was not written as it was (NaN payloads aside)
    for got, exp in ((dk.cpu(), want[0]), (dv.cpu(), want[1])):
        assert torch.equal(got[..., :512], exp[..., :512])
        assert same_bits(got[..., 512:].contiguous().view(torch.bfloat16), exp[..., 512:].contiguous().view(torch.bfloat16))
    order = order.to(torch.int32)
    rk, rv = kernels.kv4_read(dk, dv, order.to(DEV), err=err)
    assert int(err.item()) == 0
    for got, exp, key in ((rk, want[0], True), (rv, want[1], False)):
        # m + c s is one rounding away from exact in 64 bits, then one to bf16
        x = ref.values(exp[order.long()], key).float().to(torch.bfloat16)
        assert same_bits(got.cpu(), x)


def test_ties_round_to_even_codes():
    """Rows on which every (x - m) / s is a multiple of 1/2 or 1/4, over many
    scales: the codes are those of an IEEE division with ties to even."""
    from cache_eviction_b200 import kernels
    rows = []
    for e in list(range(-130, 120, 5)) + [-133]:
        for step in (1, 3, 5, 7, 129, 131, 255):
            s = step * 2.0 ** e
            for q in (2.0, 4.0):
                x = torch.arange(64, dtype=torch.float64).remainder(15 * q + 1) / q * s
                rows += [x, x - 7.5 * s, -x]
    x = torch.stack(rows).clamp(-3.38e38, 3.38e38).to(torch.bfloat16).view(-1, 1, 64)
    T = x.shape[0]
    units = -(-T // 16)
    pool = torch.zeros((2, units, 1, 576), dtype=torch.uint8, device=DEV)
    kernels.kv4_write(x.to(DEV), x.to(DEV), pool[0], pool[1], torch.arange(T, device=DEV))
    want = [t.view(-1, *t.shape[2:]) for t in ref.quantise(x)]
    for kv, key in ((0, True), (1, False)):
        got = [t.view(units * 16, -1)[:T] for t in ref.unpack(pool[kv].cpu()[:, 0], key)]
        for a, b in zip(got, want):
            assert torch.equal(a, b.double().view(T, -1))


def test_rounding_stays_within_half_a_step():
    """|x - value| <= s / 2, or 15 s 2^-8 at the top code (s rounded down by up
    to 2^-9 of itself), plus the roundings of x - m and of the value (2^-8)."""
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn((4096, 8, 64), generator=gen) * torch.exp(2 * torch.randn((4096, 8, 1), generator=gen))).to(torch.bfloat16)
    pool = torch.zeros((2, 256, 8, 576), dtype=torch.uint8, device=DEV)
    kernels.kv4_write(x.to(DEV), x.to(DEV), pool[0], pool[1], torch.arange(4096, device=DEV))
    for out in kernels.kv4_read(pool[0], pool[1], torch.arange(256, dtype=torch.int32, device=DEV)):
        got = out.transpose(1, 2).reshape(4096, 8, 64).double().cpu()
        s = ref.quantise(x)[1].double()[..., None]
        slack = s * max(0.5, 15 * 2.0 ** -8) * (1 + 2.0 ** -20) + got.abs() * 2.0 ** -8 + x.double().abs() * 2.0 ** -22
        assert ((got - x.double()).abs() <= slack).all()


def test_write_takes_views_and_skips_padding():
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(4)
    T, G, units = 37, 8, 6
    qkv = torch.randn((T, (64 + 16) * 64 + 3), generator=gen).to(torch.bfloat16).to(DEV)
    loc = torch.randperm(units * 16, generator=gen)[:T]
    loc[5], loc[6], loc[7] = -1, -2 ** 40, units * 16      # padding, padding, beyond the pool
    plain = torch.full((2, units, G, 576), 7, dtype=torch.uint8, device=DEV)
    kept = loc.clone()
    kept[7] = -1
    for a, b in ((64 * 64, 72 * 64), (64 * 64 + 3, 72 * 64 + 3)):         # aligned and odd starts
        k, v = (qkv[:, s:s + 512].view(T, G, 64) for s in (a, b))
        for kk, vv in ((k, v), (k.transpose(0, 1).contiguous().transpose(0, 1), v.flip(2).flip(2))):
            want, got = plain.clone(), plain.clone()
            err = torch.zeros(1, dtype=torch.int32, device=DEV)
            kernels.kv4_write(kk.contiguous(), vv.contiguous(), want[0], want[1], kept.to(DEV), err=err)
            assert int(err.item()) == 0
            kernels.kv4_write(kk, vv, got[0], got[1], loc.to(DEV), err=err)
            assert int(err.item()) == 1                                   # CE_EW_INDEX
            assert torch.equal(got, want)
            touched = (got != 7).any(-1).any(-1).sum()
            assert touched == 2 * len(set((loc[(loc >= 0) & (loc < units * 16)] // 16).tolist()))


def test_read_strides_and_skipped_pages():
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(5)
    G, units = 4, 9
    k, v = ref.random_pool(units, G, True, gen).to(DEV), ref.random_pool(units, G, False, gen).to(DEV)
    order = torch.tensor([3, -1, 8, 0, 3, 9], dtype=torch.int32, device=DEV)   # a repeat, padding, beyond
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    rows = torch.full((2, 6, 16, G, 72), 5.0, dtype=torch.bfloat16, device=DEV)   # token-major, padded rows
    kernels.kv4_read(k, v, order, k_out=rows[0, ..., :64].transpose(1, 2), v_out=rows[1, ..., :64].transpose(1, 2), err=err)
    assert int(err.item()) == 1
    assert (rows[..., 64:] == 5).all() and (rows[:, [1, 5]] == 5).all()
    for i, u in ((0, 3), (2, 8), (3, 0), (4, 3)):
        for kv, pool, key in ((0, k, True), (1, v, False)):
            want = ref.values(pool[u].cpu(), key).float().to(torch.bfloat16)
            assert torch.equal(rows[kv, i, ..., :64].transpose(0, 1).cpu(), want)
    a, b = kernels.kv4_read(k, v, order[:0])
    assert a.shape == b.shape == (0, G, 16, 64)


# ---------------------------------------------------------------- attention
def batch(lens, G, gen, spread=1.0, garbage=True):
    """Pools, CSR and the 64-bit per-row pages of a batch of 4-bit rows; slots
    past a row's end and unused units hold 0xff bytes (NaN scales)."""
    counts = [-(-n // 16) for n in lens]
    units = sum(counts) + 3
    pools = [ref.random_pool(units, G, key, gen, spread) for key in (True, False)]
    order = torch.randperm(units, generator=gen)[:sum(counts)]
    indptr = torch.tensor([0] + counts).cumsum(0)
    if garbage:
        used = torch.zeros((units, 16), dtype=torch.bool)
        for b, n in enumerate(lens):
            for i in range(counts[b]):
                used[order[indptr[b] + i], :max(0, min(16, n - 16 * i))] = True
        for key, pool in ((True, pools[0]), (False, pools[1])):
            byte, _ = ref.byte_of(key)
            dead = torch.zeros((units, 576), dtype=torch.bool)
            for j in range(16):
                gone = ~used[:, j]
                dead[gone[:, None] & torch.zeros(576, dtype=torch.bool).scatter(0, byte[j], True)] = True
                dead[gone, 512 + 4 * j:516 + 4 * j] = True
            pool[dead[:, None].expand(-1, G, -1)] = 255
    csr = (indptr.to(torch.int32).to(DEV), order.to(torch.int32).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    return pools[0], pools[1], csr, order, indptr


def check(lens, G, modes, seed, sinks=True, spread=1.0, qspread=1.5, zero_new=True, call=None, **kw):
    """Runs the operator over a batch and holds every output to the 64-bit form."""
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(seed)
    B, H = len(lens), 8 * G
    kp, vp, csr, order, indptr = batch(lens, G, gen, spread)
    units = kp.shape[0]
    q = (torch.randn((B, H, 64), generator=gen) * qspread).to(torch.bfloat16)
    sink = torch.randn(H, generator=gen) if sinks else None
    rows = torch.randperm(B + 2, generator=gen)[:B]
    mode = torch.zeros(B + 2, dtype=torch.int32)
    mode[rows] = torch.tensor([modes[i % len(modes)] for i in range(B)], dtype=torch.int32)
    old = torch.rand((G, units), generator=gen)
    scores, lse = old.to(DEV), torch.empty((B, H), device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    call = call or kernels.kv4_decode_attn_score
    out = call(q.to(DEV), kp.to(DEV), vp.to(DEV), *csr, SCALE, sinks=None if sink is None else sink.to(DEV),
               mode_of_row=mode.to(DEV), rows=rows.to(DEV), scores=scores, zero_new=zero_new, lse=lse, err=err, **kw)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    out, lse, scores = out.double().cpu(), lse.double().cpu(), scores.double().cpu()
    want_scores = old.double().clone()
    tol_scores = torch.zeros_like(want_scores)
    for b, n in enumerate(lens):
        u = order[indptr[b]:indptr[b + 1]]
        for g in range(G):
            hs = slice(8 * g, 8 * g + 8)
            snk = None if sink is None else sink[hs].double()
            if n == 0:
                assert (out[b, hs] == 0).all()
                assert torch.allclose(lse[b, hs], torch.full((8,), -math.inf, dtype=torch.float64) if snk is None else snk)
                continue
            (kc, ks, km), (vc, vs, vm) = ((x.reshape(-1, x.shape[-1])[:n] for x in ref.unpack(t[u, g], key))
                                          for t, key in ((kp, True), (vp, False)))
            qq = q[b, hs].double()
            p, o, l = ref.attend(qq[None], km + kc * ks, vm + vc * vs, torch.ones(1, n, dtype=torch.bool), snk, SCALE)
            p, o, l = p[0], o[0], l[0]
            d = 80 * 2.0 ** -24 * SCALE * (qq.abs() @ kc.T * ks.T + qq.abs().sum(-1, keepdim=True) * km.abs().T).amax(-1)
            logits = qq @ (km + kc * ks).T * SCALE
            e = 2 * d + 16 * 2.0 ** -24 * (1 + (logits - l[:, None]).abs().amax(-1))
            e = e[:, None]
            tol = (2.0 ** -8 * o.abs() + (2.0 ** -11 + e) * (p @ (vc * vs)) + e * (p @ vm.abs())
                   + 2.0 ** -38 * n * vs.max() * 15 + 1e-37)
            assert ((out[b, hs] - o).abs() <= tol).all(), (b, g, n, float(((out[b, hs] - o).abs() / tol).max()))
            assert ((lse[b, hs] - l).abs() <= e[:, 0] + 2.0 ** -22 * (1 + l.abs())).all()
            m = int(mode[rows[b]])
            if m:
                mass = torch.zeros(len(u) * 16, dtype=torch.float64)
                mass[:n] = p.sum(0) if m == 1 else p.amax(0)
                mass = mass.view(-1, 16).sum(-1)
                if zero_new and n % 16 == 1:
                    want_scores[g, u[-1]] = 0.0
                want_scores[g, u] += mass
                rel = e.max() + 2.0 ** -23 * (8 + l.abs().max() / math.log(2) + logits.abs().max() / math.log(2))
                tol_scores[g, u] = rel * mass + 1e-30
    tol_scores += 2.0 ** -23 * want_scores.abs()
    assert ((scores - want_scores).abs() <= tol_scores).all(), float(((scores - want_scores).abs() / tol_scores.clamp(min=1e-30)).max())
    return out


@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_decode_lengths_and_modes(G):
    check([1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 0, 511, 512, 513, 1000, 0], G, [0, 1, 2], seed=20 + G)


@pytest.mark.parametrize("n", [1, 16, 64, 517, 9001, 70003])
def test_decode_one_sequence(n):
    check([n], 8, [1], seed=n)
    check([n], 1, [2], seed=n + 1, sinks=False)


def test_decode_wide_batch():
    check([(37 * i) % 211 for i in range(400)], 2, [0, 1, 2], seed=6)


@pytest.mark.parametrize("spread,qspread", [(1e-3, 1.0), (30.0, 1.0), (1e15, 1e-15), (1.0, 1e4), (1e-30, 1e30)])
def test_decode_ranges(spread, qspread):
    """Rows far from 1 and query rows far from 1: the powers of two that keep
    both matrix products in fp16's range come and go without a trace."""
    check([700, 65, 3], 2, [1], seed=7, spread=spread, qspread=qspread)


def test_decode_scales_that_grow_along_a_row():
    """V scales that rise by powers of two page by page: the accumulators are
    rescaled many times, up to 2^60 apart."""
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(8)
    n, G = 16 * 61, 1
    x = torch.randn((61, G, 16, 64), generator=gen)
    kp = ref.pack(*ref.quantise((x * 0.01).to(torch.bfloat16)), True)
    for sign in (1, -1):
        v = (torch.randn((61, G, 16, 64), generator=gen) * 2.0 ** (sign * torch.arange(61.0) - 30).view(-1, 1, 1, 1)).to(torch.bfloat16)
        vp = ref.pack(*ref.quantise(v), False)
        q = torch.randn((1, 8, 64), generator=gen).to(torch.bfloat16)
        out = kernels.kv4_decode_attn_score(q.to(DEV), kp.to(DEV), vp.to(DEV), torch.tensor([0, 61], dtype=torch.int32, device=DEV),
                                            torch.arange(61, dtype=torch.int32, device=DEV),
                                            torch.tensor([n], dtype=torch.int32, device=DEV), SCALE)
        kk, vv = ref.values(kp, True)[:, 0].reshape(n, 64), ref.values(vp, False)[:, 0].reshape(n, 64)
        p, o, _ = ref.attend(q.double(), kk, vv, torch.ones(1, n, dtype=torch.bool), None, SCALE)
        tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 1e-5) * (p @ vv.abs()) * 2
        assert ((out.double().cpu() - o).abs() <= tol).all()


def test_decode_keeps_nan_to_its_own_heads_and_rows():
    """A visible row with a NaN makes its KV head's outputs NaN, and no other's."""
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(9)
    G, lens = 2, [100, 100]
    kp, vp, csr, order, indptr = batch(lens, G, gen)
    vp[order[3], 1, 512:516] = torch.tensor([0xc0, 0x7f, 0xc0, 0x7f], dtype=torch.uint8)   # row 0, head 1, token 48
    q = torch.randn((2, 16, 64), generator=gen).to(torch.bfloat16).to(DEV)
    out = kernels.kv4_decode_attn_score(q, kp.to(DEV), vp.to(DEV), *csr, SCALE)
    assert out[0, 8:].isnan().all() and not out[0, :8].isnan().any() and not out[1].isnan().any()


def test_decode_strides_streams_and_deferred_scores():
    from cache_eviction_b200 import capi, kernels
    lens, G = [300, 17, 1025], 8
    wide = torch.zeros((3, 70, 192), dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()

    def strided(q, *a, **kw):
        view = torch.zeros((3, 65, 130), dtype=torch.bfloat16, device=DEV)[:, 1:, 2:66]
        view.copy_(q)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = kernels.kv4_decode_attn_score(view, *a, out=wide[:, 3:67, 64:128], **kw)
        torch.cuda.current_stream().wait_stream(side)
        return out

    def deferred(q, kp, vp, indptr, indices, tokens, scale, **kw):
        need = kernels.kv4_decode_workspace_bytes(3, indices.numel(), 64, G)
        ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
        out = kernels.kv4_decode_attn_score(q, kp, vp, indptr, indices, tokens, scale, workspace=ws,
                                            score_flags=3 | capi.CE_SCORE_DEFER, **kw)
        kernels.decode_scores(indptr, indices, tokens, kp.shape[0], 16, 64, G, 3, kw["mode_of_row"], kw["rows"],
                              kw["scores"], ws, zero_new=kw["zero_new"])
        return out
    a = check(lens, G, [1, 2, 0], seed=10, call=strided)
    b = check(lens, G, [1, 2, 0], seed=10, call=deferred)
    assert torch.equal(a, b)
    assert (wide[:, :3] == 0).all() and (wide[:, :, :64] == 0).all() and (wide[:, :, 128:] == 0).all()


def test_decode_is_repeatable_and_captured_graphs_do_not_share():
    """Two graphs of different batches, captured without a workspace, replayed
    in turn and at once on two streams: each gives what the eager call gave."""
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(11)
    made = []
    for lens in ([2000, 31, 700], [64] * 9):
        kp, vp, csr, _, _ = batch(lens, 4, gen)
        q = torch.randn((len(lens), 32, 64), generator=gen).to(torch.bfloat16).to(DEV)
        a = (q, kp.to(DEV), vp.to(DEV), *csr, SCALE)
        eager = kernels.kv4_decode_attn_score(*a)
        for _ in range(3):
            assert torch.equal(kernels.kv4_decode_attn_score(*a), eager)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernels.kv4_decode_attn_score(*a)
        made.append((graph, out, eager, a))
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(20):
        for (graph, out, _, _), st in zip(made, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, eager, _ in made:
        assert torch.equal(out, eager)


def test_pools_beyond_32_bit_offsets():
    """Units whose slices lie past 4 GiB are written, read and attended to."""
    from cache_eviction_b200 import kernels
    G, units = 8, 1_000_000
    k = torch.zeros((units, G, 576), dtype=torch.uint8, device=DEV)
    v = torch.zeros((units, G, 576), dtype=torch.uint8, device=DEV)
    assert k.numel() > 2 ** 32
    gen = torch.Generator(device=DEV).manual_seed(12)
    u = torch.tensor([units - 1, 3, units - 2, 700_001], dtype=torch.int32, device=DEV)
    x = torch.randn((2, 64, G, 64), generator=gen, device=DEV).to(torch.bfloat16)
    loc = (u.long()[:, None] * 16 + torch.arange(16, device=DEV)).view(-1)
    kernels.kv4_write(x[0], x[1], k, v, loc)
    small = torch.zeros((2, 4, G, 576), dtype=torch.uint8, device=DEV)
    kernels.kv4_write(x[0], x[1], small[0], small[1], torch.arange(64, device=DEV))
    assert torch.equal(k[u.long()], small[0]) and torch.equal(v[u.long()], small[1])
    ident = torch.arange(4, dtype=torch.int32, device=DEV)
    for a, b in zip(kernels.kv4_read(k, v, u), kernels.kv4_read(small[0], small[1], ident)):
        assert torch.equal(a, b)
    q = torch.randn((1, 64, 64), generator=gen, device=DEV).to(torch.bfloat16)
    indptr, tokens = torch.tensor([0, 4], dtype=torch.int32, device=DEV), torch.tensor([61], dtype=torch.int32, device=DEV)
    assert torch.equal(kernels.kv4_decode_attn_score(q, k, v, indptr, u, tokens, SCALE),
                       kernels.kv4_decode_attn_score(q, small[0], small[1], indptr, ident, tokens, SCALE))


def test_bad_units_are_flagged_and_skipped():
    from cache_eviction_b200 import capi, kernels
    gen = torch.Generator().manual_seed(13)
    kp, vp, (indptr, indices, tokens), _, _ = batch([100, 40], 8, gen)
    q = torch.randn((2, 64, 64), generator=gen).to(torch.bfloat16).to(DEV)
    a = (q, kp.to(DEV), vp.to(DEV))
    good = kernels.kv4_decode_attn_score(*a, indptr, indices, tokens, SCALE)
    for bad in (-5, kp.shape[0], 2 ** 31 - 1):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        idx = indices.clone()
        idx[2] = bad
        out = kernels.kv4_decode_attn_score(*a, indptr, idx, tokens, SCALE, err=err)
        assert int(err.item()) == capi.CE_EW_INDEX
        assert torch.equal(out[1], good[1])           # the other row is untouched by it
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    kernels.kv4_decode_attn_score(*a, indptr, indices[:8].contiguous(), tokens, SCALE, err=err)
    assert int(err.item()) == capi.CE_EW_CAPACITY
