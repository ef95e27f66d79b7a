"""Windowed attention on the GPU (ce_window_decode, ce_window_prefill) against
the same mask in 64 bits.

Tolerances per value, from the arithmetic: logits are fp32 sums of 64 exact
bf16 products, off by at most d = 80 * 2^-24 * scale * sum |q k|; a p is off by
at most the relative e = 2 d + 16 * 2^-24 * (1 + |logit range|).  The decode form
splits p into two bf16 parts (2^-17), so |error| <= (2^-17 + e) sum p |v| plus the
output's rounding (2^-8 in bf16, 2^-24 in fp32).  The prefill form rounds p to
bf16 (2^-8 of each): |error| <= (2^-8 + e) sum p |v| + 2^-8 |o|.
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


def batch(lens, G, P, gen, garbage=float("nan")):
    """Scattered bf16 pages of a batch; every slot that holds no token of a row
    holds `garbage`."""
    counts = [-(-n // P) for n in lens]
    units = sum(counts) + 3
    order = torch.randperm(units, generator=gen)[:sum(counts)]
    indptr = torch.tensor([0] + counts).cumsum(0)
    pools = torch.full((2, units, G, P, 64), garbage, dtype=torch.bfloat16)
    flat = []
    for b, n in enumerate(lens):
        x = (torch.randn((2, n, G, 64), generator=gen) + 0.3 * torch.randn((2, 1, G, 64), generator=gen)).to(torch.bfloat16)
        flat.append(x)
        t = torch.arange(n)
        u = order[indptr[b] + t // P]
        pools[:, u, :, t % P] = x.transpose(0, 1)
    csr = (indptr.to(torch.int32).to(DEV), order.to(torch.int32).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    return pools, flat, csr, order, indptr


def visible(pos, n, window, first):
    """[len(pos), n] mask of the definition."""
    t = torch.arange(n)[None]
    m = t <= pos[:, None]
    return m & ((t > pos[:, None] - window) | (t < first)) if window >= 0 else m


def hold(got, q, k, v, seen, sink, bf16_p, lse=None, f32=False):
    """got [n, 8, 64] of one KV head against the 64-bit form."""
    if k.shape[0] == 0:      # nothing but the sink
        assert (got == 0).all()
        want = torch.full((8,), -math.inf) if sink is None else sink
        assert lse is None or torch.allclose(lse.double()[0], want.double(), rtol=2.0 ** -22, atol=2.0 ** -22)
        return
    q, k, v = q.double(), k.double(), v.double()
    p, o, l = ref.attend(q, k, v, seen, sink, SCALE)
    d = 80 * 2.0 ** -24 * SCALE * torch.einsum("njd,td->njt", q.abs(), k.abs())
    d = torch.where(seen[:, None], d, 0.0).amax(-1)
    z = torch.einsum("njd,td->njt", q, k) * SCALE
    span = torch.where(seen[:, None], (z - l[..., None]).abs(), 0.0).amax(-1)
    e = 2 * d + 16 * 2.0 ** -24 * (1 + span)
    e = torch.where(l.isinf(), 0.0, e)[..., None]
    w = 2.0 ** -8 if bf16_p else 2.0 ** -17
    tol = (w + e) * torch.einsum("njt,td->njd", p, v.abs()) + (2.0 ** -24 if f32 else 2.0 ** -8) * o.abs() + 1e-30
    bad = ((got.double() - o).abs() / tol)
    assert not got.isnan().any() and (bad <= 1).all(), float(bad.nan_to_num(1e9).max())
    if lse is not None:
        ok = torch.where(l.isinf(), lse.double() == l, (lse.double() - l).abs() <= e[..., 0] + 2.0 ** -22 * (1 + l.abs()))
        assert ok.all()


# ------------------------------------------------------------ single tokens
def check_step(lens, G, P, window, first, seed, sinks=True, call=None, **kw):
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(seed)
    B, H = len(lens), 8 * G
    pools, flat, csr, order, indptr = batch(lens, G, P, gen)
    if window >= 0:     # what the mask hides may hold anything, in pages that are partly visible too
        for b, n in enumerate(lens):
            t = torch.arange(n)
            t = t[~visible(torch.tensor([n - 1]), n, window, first)[0]]
            bad = torch.tensor([math.nan, math.inf, -math.inf, -3.3895e38])[t % 4].to(torch.bfloat16)
            pools[:, order[indptr[b] + t // P], :, t % P] = bad.view(-1, 1, 1, 1)
    q = (torch.randn((B, H, 64), generator=gen) * 1.5).to(torch.bfloat16)
    sink = torch.randn(H, generator=gen) if sinks else None
    err, lse = torch.zeros(1, dtype=torch.int32, device=DEV), torch.empty((B, H), device=DEV)
    out = (call or kernels.window_decode)(q.to(DEV), pools[0].to(DEV), pools[1].to(DEV), *csr, SCALE, P, window, first=first,
                                          sinks=None if sink is None else sink.to(DEV), lse=lse, err=err, **kw)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    for b, n in enumerate(lens):
        seen = visible(torch.tensor([n - 1]), n, window, first)
        for g in range(G):
            hs = slice(8 * g, 8 * g + 8)
            hold(out[b:b + 1, hs].cpu(), q[b:b + 1, hs], flat[b][0][:, g], flat[b][1][:, g], seen,
                 None if sink is None else sink[hs].double(), False, lse[b:b + 1, hs].cpu(), out.dtype == torch.float32)
    return out


LENS = [1, 2, 15, 16, 17, 31, 100, 127, 128, 129, 0, 255, 257, 511, 700, 1000, 0]


@pytest.mark.parametrize("G,P", [(1, 16), (2, 16), (4, 16), (8, 16), (8, 1)])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (16, 0), (17, 3), (128, 0), (100, 16), (130, 129), (513, 40),
                                          (1, 600), (2 ** 31 - 1, 2 ** 31 - 1), (-1, 0), (-1, 5)])
def test_step_masks(G, P, window, first):
    check_step(LENS, G, P, window, first, seed=G + P + window % 97)


@pytest.mark.parametrize("n,window,first", [(20011, 4099, 5), (20011, 6000, 2048), (50000, 128, 0), (1, 1, 0)])
def test_step_one_sequence(n, window, first):
    check_step([n], 8, 16, window, first, seed=n)
    check_step([n], 1, 16, window, first, seed=n, sinks=False, out_f32=True)


def test_step_without_a_window_is_the_plain_decode():
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(3)
    pools, _, csr, _, _ = batch([300, 17, 2000, 0, 64], 4, 16, gen)
    q = torch.randn((5, 32, 64), generator=gen).to(torch.bfloat16).to(DEV)
    a = (q, pools[0].to(DEV), pools[1].to(DEV), *csr, SCALE, 16)
    want = kernels.decode_attn_score(*a, score_flags=0)
    for window, first in ((-1, 0), (2000, 0), (5000, 7), (1, 5000)):
        assert torch.equal(kernels.window_decode(*a, window, first=first), want)


def test_step_strides_stream_and_graph():
    from cache_eviction_b200 import kernels
    side = torch.cuda.Stream()
    wide = torch.zeros((3, 70, 192), dtype=torch.bfloat16, device=DEV)

    def strided(q, *a, **kw):
        view = torch.zeros((3, 65, 131), dtype=torch.bfloat16, device=DEV)[:, 1:, 3:67]     # odd strides: copied
        view.copy_(q)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = kernels.window_decode(view, *a, out=wide[:, 3:67, 64:128], **kw)
        torch.cuda.current_stream().wait_stream(side)
        return out

    def captured(q, *a, **kw):
        kernels.window_decode(q, *a, **kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernels.window_decode(q, *a, **kw)
        out.zero_()
        graph.replay()
        return out
    a = check_step([300, 17, 1025], 8, 16, 200, 20, seed=10, call=strided)
    b = check_step([300, 17, 1025], 8, 16, 200, 20, seed=10, call=captured)
    assert torch.equal(a, b)
    assert (wide[:, :3] == 0).all() and (wide[:, :, :64] == 0).all() and (wide[:, :, 128:] == 0).all()


# ------------------------------------------------------------------- chunks
def check_chunk(parts, G, P, window, first, seed, sinks=True, call=None, plant=None, spread=1.0, pad=2, loose=0):
    """parts: (queries, prefix) of every entry.  `pad` rows of q belong to no entry."""
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(seed)
    H = 8 * G
    lens, nqs = [a + b for a, b in parts], [a for a, _ in parts]
    pools, flat, csr, order, indptr = batch(lens, G, P, gen)
    ptr = torch.tensor([0] + nqs).cumsum(0)
    total = int(ptr[-1]) + pad
    q = (torch.randn((total, H, 64), generator=gen) * 1.5 * spread).to(torch.bfloat16)
    if plant is not None:
        plant(pools, flat, order, indptr)
    sink = torch.randn(H, generator=gen) if sinks else None
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full((total, H, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    out = (call or kernels.window_prefill)(q.to(DEV), pools[0].to(DEV), pools[1].to(DEV), ptr.to(torch.int32).to(DEV), *csr, SCALE, P,
                                           max(nqs) + loose, max(lens) + loose, window, first=first,
                                           sinks=None if sink is None else sink.to(DEV), err=err, out=out)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    got = out.cpu()
    assert (got[int(ptr[-1]):] == 7).all()           # rows of no entry
    for b, (nq, pre) in enumerate(parts):
        if nq == 0:
            continue
        seen = visible(torch.arange(pre, pre + nq), pre + nq, window, first)
        for g in range(G):
            hs = slice(8 * g, 8 * g + 8)
            k, v = flat[b][0][:, g], flat[b][1][:, g]
            rows = torch.arange(nq)
            if plant is not None:       # rows that see a planted value are NaN, the others as if it were not there
                bad = ~(torch.isfinite(v).all(-1) & torch.isfinite(k).all(-1))
                hit = (seen & bad).any(-1)
                assert not torch.isfinite(got[ptr[b]:ptr[b + 1], hs][hit]).all(-1).any()
                rows = rows[~hit]
                k, v = (torch.where(bad[:, None], 0.0, x.float()).to(torch.bfloat16) for x in (k, v))
            if len(rows):
                hold(got[ptr[b]:ptr[b + 1], hs][rows], q[ptr[b]:ptr[b + 1], hs][rows], k, v, seen[rows],
                     None if sink is None else sink[hs].double(), True)
    return out


MASKS = [(1, 0), (1, 1), (16, 0), (17, 3), (128, 0), (100, 16), (130, 129), (300, 40), (1, 600), (140, 300),
         (2 ** 31 - 1, 2 ** 31 - 1), (-1, 0), (-1, 5)]


@pytest.mark.parametrize("window,first", MASKS)
@pytest.mark.parametrize("G,P", [(1, 16), (8, 16), (2, 8), (1, 32), (3, 64), (2, 1), (1, 4)])
def test_chunk_masks(G, P, window, first):
    check_chunk([(1, 0), (15, 0), (16, 5), (17, 100), (0, 3), (33, 127), (128, 128), (150, 300), (40, 613)], G, P, window, first,
                seed=G * 100 + P + window % 97)


@pytest.mark.parametrize("nq,pre,window,first", [(1, 9000, 300, 20), (1000, 5000, 1024, 256), (2049, 0, 128, 0), (513, 7, -1, 0),
                                                 (257, 8191, 6144, 2048), (64, 20000, -1, 0)])
def test_chunk_long(nq, pre, window, first):
    check_chunk([(nq, pre)], 1, 16, window, first, seed=nq + pre, sinks=nq % 2 == 0, loose=50)


@pytest.mark.parametrize("spread", [1e-3, 30.0, 1000.0])
def test_chunk_logit_ranges(spread):
    """From a nearly uniform softmax to one key per row: maxima that rise by
    more than 2^8 from tile to tile rescale the accumulators."""
    check_chunk([(100, 900)], 2, 16, -1, 0, seed=5, spread=spread)
    check_chunk([(100, 900)], 2, 16, 500, 100, seed=6, spread=spread)


@pytest.mark.parametrize("P", [16, 1])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_chunk_values_that_are_not_finite_reach_only_who_sees_them(P, bad):
    """Planted in the chunk (later queries see them), in the window's edge and
    between the first tokens and the window, in one value or a whole row."""
    def plant(pools, flat, order, indptr):
        for kv, b, t, g, dims in ((1, 0, 620, 0, slice(0, 64)), (1, 0, 627, 1, slice(9, 10)), (1, 0, 430, 0, slice(63, 64)),
                                  (1, 0, 200, 0, slice(0, 64)), (1, 1, 3, 1, slice(0, 1)), (1, 1, 4, 0, slice(0, 64)),
                                  (0, 0, 500, 1, slice(0, 64)), (0, 1, 30, 0, slice(0, 64))):
            flat[b][kv, t, g, dims] = bad
            pools[kv, order[indptr[b] + t // P], g, t % P, dims] = bad
    check_chunk([(60, 600), (50, 0)], 2, P, 180, 20, seed=7, plant=plant)
    check_chunk([(60, 600), (50, 0)], 2, P, -1, 0, seed=8, plant=plant)


def test_chunk_masked_extremes_do_not_leak():
    """Hidden values of the largest magnitude: a weight that is only nearly 0 would show."""
    from cache_eviction_b200 import kernels
    hot = [640, 655, 300, 410]
    seen = visible(torch.arange(600, 660), 660, 180, 20)[:, hot].any(-1)
    assert seen.any() and not seen.all()

    def call(q, k, v, qo, indptr, indices, tokens, *a, out=None, **kw):
        clean = kernels.window_prefill(q, k, v, qo, indptr, indices, tokens, *a, out=out.clone(), **kw)
        for t in hot:
            v[indices[t // 16].long(), :, t % 16] = 3.3895e38
        planted = kernels.window_prefill(q, k, v, qo, indptr, indices, tokens, *a, out=out.clone(), **kw)
        assert torch.equal(planted[:60][~seen.to(DEV)], clean[:60][~seen.to(DEV)])
        assert not torch.equal(planted, clean)
        return clean
    check_chunk([(60, 600)], 1, 16, 180, 20, seed=9, call=call)


def test_chunk_of_single_tokens_is_the_step():
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(11)
    lens = [1, 40, 333, 2000]
    pools, _, csr, _, _ = batch(lens, 4, 16, gen)
    q = torch.randn((4, 32, 64), generator=gen).to(torch.bfloat16).to(DEV)
    a = (pools[0].to(DEV), pools[1].to(DEV))
    one = torch.arange(5, dtype=torch.int32, device=DEV)
    for window, first in ((64, 4), (-1, 0)):
        x = kernels.window_decode(q, *a, *csr, SCALE, 16, window, first=first).float()
        y = kernels.window_prefill(q, *a, one, *csr, SCALE, 16, 1, 2000, window, first=first).float()
        assert float((x - y).norm() / x.norm()) < 2.0 ** -8 + 2.0 ** -8      # each within its own rounding of P and output


def test_chunk_strides_stream_and_graph():
    from cache_eviction_b200 import kernels
    side = torch.cuda.Stream()
    parts = [(40, 300), (17, 0), (100, 1025)]
    wide = torch.zeros((159, 70, 128), dtype=torch.bfloat16, device=DEV)

    def strided(q, *a, out=None, **kw):
        odd = torch.zeros((159, 65, 131), dtype=torch.bfloat16, device=DEV)[:, 1:, 3:67]     # copied
        odd.copy_(q)
        side.wait_stream(torch.cuda.current_stream())
        wide[157:, 3:67, :64] = 7
        with torch.cuda.stream(side):
            o = kernels.window_prefill(odd, *a, out=wide[:, 3:67, :64], **kw)
        torch.cuda.current_stream().wait_stream(side)
        return o

    def captured(q, *a, out=None, **kw):
        view = torch.zeros((159, 66, 72), dtype=torch.bfloat16, device=DEV)[:, 2:, 8:]       # taken as it is
        view.copy_(q)
        kernels.window_prefill(view, *a, out=out, **kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kernels.window_prefill(view, *a, out=out, **kw)
        out[:157].zero_()
        graph.replay()
        return out
    a = check_chunk(parts, 8, 16, 200, 20, seed=10, call=strided)
    b = check_chunk(parts, 8, 16, 200, 20, seed=10, call=captured)
    assert torch.equal(a, b)
    assert (wide[:, :3] == 0).all() and (wide[:, :, 64:] == 0).all()


def test_chunk_bad_entries_are_flagged_and_left():
    from cache_eviction_b200 import capi, kernels
    gen = torch.Generator().manual_seed(12)
    pools, _, csr, _, _ = batch([50, 60], 1, 16, gen)
    q = torch.randn((30, 8, 64), generator=gen).to(torch.bfloat16).to(DEV)
    a = (q, pools[0].to(DEV), pools[1].to(DEV))
    qo = torch.tensor([0, 10, 30], dtype=torch.int32, device=DEV)
    good = kernels.window_prefill(*a, qo, *csr, SCALE, 16, 20, 60, 30)

    def run(qo=qo, csr=csr, max_q=20, max_tokens=60):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = torch.full_like(q, 3.0)
        kernels.window_prefill(*a, qo, *csr, SCALE, 16, max_q, max_tokens, 30, err=err, out=out)
        return int(err.item()), out
    flag, out = run(max_q=19)                                   # the second chunk is longer than the bound
    assert flag == capi.CE_EW_SHAPE and torch.equal(out[:10], good[:10]) and (out[10:] == 3).all()
    flag, out = run(max_tokens=59)
    assert flag == capi.CE_EW_SHAPE and torch.equal(out[:10], good[:10]) and (out[10:] == 3).all()
    flag, out = run(qo=torch.tensor([0, 10, 31], dtype=torch.int32, device=DEV))
    assert flag == capi.CE_EW_SHAPE and (out[10:] == 3).all()
    flag, out = run(csr=(csr[0], csr[1][:6].contiguous(), csr[2]))   # the list is cut short
    assert flag == capi.CE_EW_SHAPE and torch.equal(out[:10], good[:10]) and (out[10:] == 3).all()
    idx = csr[1].clone()
    idx[5] = pools.shape[1]
    flag, out = run(csr=(csr[0], idx, csr[2]))
    assert flag == capi.CE_EW_INDEX and torch.equal(out[:10], good[:10])


@pytest.mark.parametrize("G,lens", [(1, [33, 16, 17, 1, 0, 64, 15]), (8, [600, 31, 0, 601]), (2, [2400, 7])])
def test_chunk_items_of_pairs_and_single_tiles(G, lens):
    """Batches whose query tiles are all single ones, whole rounds of pairs, and
    pairs with a last round of single ones, with empty entries among them."""
    check_chunk([(n, 40 * (i % 3)) for i, n in enumerate(lens)], G, 16, 50, 4, seed=91 + G)


def test_chunk_is_repeatable_on_two_streams_at_once():
    """Many items per CTA, replayed from two captured graphs on two streams:
    every run gives the same bits."""
    from cache_eviction_b200 import kernels
    gen = torch.Generator().manual_seed(17)
    made = []
    for parts, G, window, first in (([(700, 60), (33, 500), (1, 0), (0, 9), (1200, 0)], 8, 100, 20), ([(300, 2000)], 2, -1, 0)):
        pools, _, csr, _, _ = batch([a + b for a, b in parts], G, 16, gen)
        nqs = [a for a, _ in parts]
        ptr = torch.tensor([0] + nqs).cumsum(0).to(torch.int32).to(DEV)
        q = torch.randn((sum(nqs), 8 * G, 64), generator=gen).to(torch.bfloat16).to(DEV)
        a = (q, pools[0].to(DEV), pools[1].to(DEV), ptr, *csr, SCALE, 16, max(nqs), max(a + b for a, b in parts), window)
        want = kernels.window_prefill(*a, first=first)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernels.window_prefill(*a, first=first)
        made.append((graph, out, want, a))
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(40):
        for (graph, out, _, _), st in zip(made, streams):
            with torch.cuda.stream(st):
                out.fill_(math.nan)
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in made:
            assert torch.equal(out, want)
