"""The ragged decode engine over 4-bit pages (kv_bits=4).

A bf16 engine runs in lockstep over the values of the same pages: its pools are
the 4-bit pools read back, its scores are copied from the 4-bit engine before
every step, so both take the same boundaries.  Then tables, positions, counts,
freed units and scores have to be equal bit for bit, and so do the 4-bit pools
read back and the bf16 pools that moved with them.  Outputs are held to
attention over the 4-bit pages in 64 bits, with the tolerances of the operator:
a logit is off by at most d = 80 * 2^-24 * scale * (s sum |q| c + |m| sum |q|), a p
by the relative e = 2 d + 16 * 2^-24 * (1 + |logit range|), p s is rounded to fp16
(2^-11, and 2^-38 of the largest below its normal range), the output to bf16.
"""
import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
L, H, G, P = 2, 64, 8, 16
STEPS = 6
SCALE = 0.125


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from cache_eviction_b200 import capi
    capi.load()


def _specs():
    from cache_eviction_b200.policy import EvictionConfig, sweep_split

    def cfg(name, budget, seed):
        p, r = sweep_split(budget, name)
        return EvictionConfig(name, budget, p, r, seed=seed)
    return [dict(ctx=4094, cfg=cfg("head_sum_2048", 2048, 1)),      # first boundary at 4,096
            dict(ctx=6142, cfg=cfg("h2o_global_2048", 2048, 2)),    # evicted; next at 6,144
            dict(ctx=5000, cfg=cfg("head_max_sum_2048", 2048, 3)),
            dict(ctx=8191, cfg=cfg("random_2048", 4096, 4)),        # boundary at 8,192
            dict(ctx=40, cfg=None),
            dict(ctx=6140, cfg=cfg("random_reservoir_2048", 2048, 5))]


def _engine(bits, overlap=False, hazard_bytes=512 << 20):
    from cache_eviction_b200.engine import RaggedDecodeEngine, synth_state
    specs = _specs()
    units = sum(-(-(sp["ctx"] + STEPS) // P) for sp in specs) + 64
    width = -(-(max(sp["ctx"] for sp in specs) + STEPS + 4096) // P)
    eng = RaggedDecodeEngine(layers=L, q_heads=H, kv_heads=G, page_size=P, pool_units=units,
                             max_rows=len(specs), r2u_width=width, pos_cap=512, device=DEV,
                             overlap_scores=overlap, kv_bits=bits, hazard_bytes=hazard_bytes)
    synth_state(eng, specs, seed=5)
    torch.cuda.synchronize()
    return eng


def _read(eng, layer):
    from cache_eviction_b200 import kernels
    return kernels.kv4_read(eng.k[layer], eng.v[layer], torch.arange(eng.units, dtype=torch.int32, device=DEV), err=eng.err)


def _hold_outputs(eng, layer, q, sink, out):
    kp, vp = eng.k[layer].cpu(), eng.v[layer].cpu()
    indptr, indices, tokens = eng.kv_indptr.cpu(), eng.kv_indices.cpu().long(), eng.kv_tokens.cpu()
    for b in range(len(eng.active)):
        u, n = indices[indptr[b]:indptr[b + 1]], int(tokens[b])
        for g in range(G):
            hs = slice(8 * g, 8 * g + 8)
            (kc, ks, km), (vc, vs, vm) = ((x.reshape(-1, x.shape[-1])[:n] for x in ref.unpack(t[u, g], key))
                                          for t, key in ((kp, True), (vp, False)))
            qq = q[b, hs].double()
            p, o, l = ref.attend(qq[None], km + kc * ks, vm + vc * vs, torch.ones(1, n, dtype=torch.bool),
                                 sink[hs].double(), SCALE)
            p, o, l = p[0], o[0], l[0]
            d = 80 * 2.0 ** -24 * SCALE * (qq.abs() @ kc.T * ks.T + qq.abs().sum(-1, keepdim=True) * km.abs().T).amax(-1)
            logits = qq @ (km + kc * ks).T * SCALE
            e = (2 * d + 16 * 2.0 ** -24 * (1 + (logits - l[:, None]).abs().amax(-1)))[:, None]
            tol = (2.0 ** -8 * o.abs() + (2.0 ** -11 + e) * (p @ (vc * vs)) + e * (p @ vm.abs())
                   + 2.0 ** -38 * n * vs.max() * 15 + 1e-37)
            assert ((out[b, hs].double() - o).abs() <= tol).all(), (b, g)


@pytest.mark.parametrize("hazard_bytes", [512 << 20, 1])      # whole batches, and a row and a layer at a time
def test_steps_and_boundaries_move_the_same_pages_as_bf16(hazard_bytes):
    a, b = _engine(4, hazard_bytes=hazard_bytes), _engine(16, hazard_bytes=hazard_bytes)
    for l in range(L):
        b.k[l], b.v[l] = (t.clone() for t in _read(a, l))
    from cache_eviction_b200 import kernels
    b.kptr, b.vptr = kernels.layer_pointers(b.k, DEV), kernels.layer_pointers(b.v, DEV)
    B = len(a.active)
    gen = torch.Generator(device=DEV).manual_seed(9)
    sinks = [torch.randn(H, generator=gen, device=DEV) for _ in range(L)]
    out = torch.empty((L, B, H, 64), dtype=torch.bfloat16, device=DEV)
    out16 = torch.empty_like(out)
    for step in range(STEPS):
        q = torch.randn((L, B, H, 64), generator=gen, device=DEV).to(torch.bfloat16)
        new = torch.randn((L, 2, B, G, 64), generator=gen, device=DEV).to(torch.bfloat16)
        b.scores.copy_(a.scores)
        slots = []

        def write(l):
            if not slots:
                slots.append(a.slots())
            a.write_layer(l, new[l, 0], new[l, 1], slots[0])
        a.step(q, out, sinks, SCALE, before_layer=write)

        def write16(l):          # what the 4-bit pool reads back as
            s = b.slots()
            assert torch.equal(s, slots[0])
            k, v = _read(a, l)
            b.write_layer(l, k[s // P, :, s % P], v[s // P, :, s % P], s)
        b.step(q, out16, sinks, SCALE, before_layer=write16)
        torch.cuda.synchronize()
        for key in ("table", "pos", "r2u", "count", "frontier", "free_stack", "free_top_dev", "kv_indptr", "kv_tokens"):
            assert torch.equal(getattr(a, key), getattr(b, key)), (step, key)
        for l in range(L):
            for x, y in zip(_read(a, l), (b.k[l], b.v[l])):
                assert torch.equal(x.view(torch.int16), y.view(torch.int16)), (step, l)
    for l in range(L):
        _hold_outputs(a, l, q[l].cpu(), sinks[l].cpu(), out[l].cpu())
    a.check_errors()
    b.check_errors()
    events = [e for r in a.active for e in a.rows[r].events]
    assert sum(e["status"] == 0 for e in events) >= 3, events
    assert events == [e for r in b.active for e in b.rows[r].events]


def test_overlapped_scores_match_inline_scores():
    """The deferred launch sums the same page log-masses against the same
    normalisers as the inline one, in another order and with another exp2: per
    page 8 exponentials (MAX: 16 of the largest) off by at most 2^-22 each and
    15 roundings of 2^-24 on either side, one more for the addition, all of
    positive terms: less than 2^-19 of the score.  Both engines start each
    step from the same scores, so that their boundaries cannot differ."""
    a, b = _engine(4, overlap=True), _engine(4)
    B = len(a.active)
    gen = torch.Generator(device=DEV).manual_seed(9)
    sinks = [torch.randn(H, generator=gen, device=DEV) for _ in range(L)]
    out_a = torch.empty((L, B, H, 64), dtype=torch.bfloat16, device=DEV)
    out_b = torch.empty_like(out_a)
    for _ in range(STEPS):
        q = torch.randn((L, B, H, 64), generator=gen, device=DEV).to(torch.bfloat16)
        b.scores.copy_(a.scores)
        a.step(q, out_a, sinks, SCALE)
        b.step(q, out_b, sinks, SCALE)
        a.join_scores()
        torch.cuda.synchronize()
        assert torch.equal(out_a, out_b)
        assert ((a.scores - b.scores).abs() <= 2.0 ** -19 * b.scores).all()
    a.check_errors()
    for key in ("table", "pos", "r2u", "count", "frontier"):
        assert torch.equal(getattr(a, key), getattr(b, key)), key
    assert a.scores.abs().sum() > 0


def test_a_step_captured_into_a_graph():
    """Write, decode and advance replayed as one graph equal the eager steps."""
    a, b = _engine(4), _engine(4)
    B = len(a.active)
    gen = torch.Generator(device=DEV).manual_seed(11)
    sinks = [torch.randn(H, generator=gen, device=DEV) for _ in range(L)]
    q = torch.randn((L, B, H, 64), generator=gen, device=DEV).to(torch.bfloat16)
    new = torch.randn((L, 2, B, G, 64), generator=gen, device=DEV).to(torch.bfloat16)
    outs = [torch.empty((L, B, H, 64), dtype=torch.bfloat16, device=DEV) for _ in range(2)]

    def body(eng, out):
        eng.advance_device()
        eng.fill()
        s = eng.slots()
        for l in range(L):
            eng.write_layer(l, new[l, 0], new[l, 1], s)
            eng.decode_layer(l, q[l], out[l], sinks[l], SCALE)
    for eng, out in ((a, outs[0]), (b, outs[1])):     # the first step sizes the workspace
        eng.advance_host()
        eng._ensure_capacity(STEPS)
        body(eng, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body(a, outs[0])
    for _ in range(3):
        new.normal_(generator=gen)
        a.advance_host()
        graph.replay()
        b.advance_host()
        body(b, outs[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
    a.check_errors()
    assert torch.equal(a.scores, b.scores) and torch.equal(a.seq_lens_dev, b.seq_lens_dev)
    for l in range(L):
        assert torch.equal(a.k[l], b.k[l]) and torch.equal(a.v[l], b.v[l])


def test_a_prompt_in_chunks_then_decode_over_4_bit_pages():
    """As a server runs them: a prompt's chunks attend to the pages read back
    so far (window_prefill), each chunk's rows are quantised into their pages,
    then a token is decoded from them."""
    from cache_eviction_b200 import kernels
    gen = torch.Generator(device=DEV).manual_seed(3)
    Gs, n, chunk = 2, 301, 96
    Hs, units = 8 * Gs, 32
    k, v = (torch.randn((n + 1, Gs, 64), generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((n + 1, Hs, 64), generator=gen, device=DEV).to(torch.bfloat16)
    kp, vp = kernels.kv4_pool(units, Gs, DEV), kernels.kv4_pool(units, Gs, DEV)
    kp.fill_(255)
    vp.fill_(255)
    pages = torch.randperm(units, generator=gen, device=DEV).to(torch.int32)[:-(-(n + 1) // P)].contiguous()
    t = torch.arange(n + 1, device=DEV)
    loc = pages.long()[t // P] * P + t % P
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    got = []
    for at in range(0, n, chunk):
        m = min(chunk, n - at)
        kernels.kv4_write(k[at:at + m], v[at:at + m], kp, vp, loc[at:at + m].contiguous(), err=err)
        have = -(-(at + m) // P)
        k16, v16 = kernels.kv4_read(kp, vp, pages[:have], err=err)
        got.append(kernels.window_prefill(q[at:at + m], k16, v16, i32(0, m), i32(0, have),
                                          torch.arange(have, dtype=torch.int32, device=DEV), i32(at + m), SCALE, P, m, at + m,
                                          100, first=7, err=err))
    kernels.kv4_write(k[n:], v[n:], kp, vp, loc[n:].contiguous(), err=err)
    last = kernels.kv4_decode_attn_score(q[n:], kp, vp, i32(0, pages.numel()), pages, i32(n + 1), SCALE, err=err)
    assert int(err.item()) == 0
    got = torch.cat(got).double().cpu()
    stored = [ref.values(ref.pack(*ref.quantise(x.cpu().view(1, -1, Gs, 64).transpose(1, 2)[0].reshape(Gs, -1, 1, 64)
                                                .expand(-1, -1, 16, -1)), key), key)[:, :, 0] for x, key in ((k, True), (v, False))]
    pos, key = torch.arange(n + 1)[:, None], torch.arange(n + 1)[None]
    seen = (key <= pos) & ((key > pos - 100) | (key < 7))
    seen[n] = True
    for g in range(Gs):
        hs = slice(8 * g, 8 * g + 8)
        kk, vv = stored[0][g], stored[1][g]
        # the chunks saw the stored values in bf16 (2^-8 of each): a logit moves by at most scale sum |q k| 2^-8
        kb, vb = (x.float().to(torch.bfloat16).double() for x in (kk, vv))
        qq = q[:, hs].double().cpu()
        p, o, _ = ref.attend(qq, kb, vb, seen, None, SCALE)
        d = 80 * 2.0 ** -24 * SCALE * torch.einsum("njd,td->njt", qq.abs(), kb.abs()).amax(-1, keepdim=True)
        e = 2 * d + 16 * 2.0 ** -24 * 100
        tol = (2.0 ** -8 + e) * torch.einsum("njt,td->njd", p, vb.abs()) + 2.0 ** -8 * o.abs()
        assert ((got[:, hs] - o[:n]).abs() <= tol[:n]).all()
        p, o, _ = ref.attend(qq[n:], kk, vv, seen[n:], None, SCALE)
        # the operator's bound, with p s c <= p (|value| + |m|) and |m| <= the largest |value|
        big = torch.einsum("njt,t->nj", p, vv.abs().amax(-1))[..., None] * 2
        tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 3 * e[n:]) * big + 1e-6
        assert ((last[0, hs].double().cpu() - o[0]).abs() <= tol[0]).all()


def test_refusals():
    from cache_eviction_b200 import capi, kernels
    from cache_eviction_b200.engine import RaggedDecodeEngine
    a = dict(layers=1, q_heads=8, kv_heads=1, pool_units=8, max_rows=1, r2u_width=8, pos_cap=8, device=DEV)
    with pytest.raises(ValueError, match="kv_bits"):
        RaggedDecodeEngine(page_size=16, kv_bits=8, **a)
    with pytest.raises(ValueError, match="16 tokens"):
        RaggedDecodeEngine(page_size=1, kv_bits=4, **a)
    with pytest.raises(capi.CeError, match="kv_bits"):
        kernels.reserve_boundary(DEV, 1, 1, 1, 16, 8, 8, 0, 1 << 20, kv_bits=8)


def test_small_decoder_with_4_bit_pages_follows_the_bf16_one():
    """OssDecoder(kv_bits=4): eager and graph steps agree bit for bit, and after
    one token the first full layer's page (the layer before it is a
    sliding-window one, kept in bf16, so both decoders give it the same rows)
    holds what the format makes of the bf16 decoder's row."""
    from cache_eviction_b200 import kernels, oss20b
    cfg = oss20b.OssConfig(layers=4, hidden=256, experts=8, top_k=2, inter=128, vocab=1000, window=16)
    w = oss20b.OssWeights(cfg, DEV, seed=5)
    prompt = torch.randint(0, cfg.vocab, (40,), generator=torch.Generator().manual_seed(6)).to(DEV)
    runs = [oss20b.OssDecoder(w, None, max_len=64, kv_bits=4) for _ in range(2)]
    plain = oss20b.OssDecoder(w, None, max_len=64)
    for dec in runs + [plain]:
        dec.tok.copy_(prompt[:1])
    for i in range(prompt.numel()):
        if i == 2:
            runs[1].capture()
        for dec in runs + [plain]:
            dec.step(prompt[i + 1:i + 2] if i + 1 < prompt.numel() else None)
        torch.cuda.synchronize()
        assert torch.equal(runs[0].logits, runs[1].logits)
        if i == 0:
            unit = int(plain.eng.r2u[0, 0])
            assert unit == int(runs[0].eng.r2u[0, 0])
            got = kernels.kv4_read(runs[0].eng.k[0], runs[0].eng.v[0], torch.tensor([unit], dtype=torch.int32, device=DEV))
            for x, full, key in ((got[0], plain.eng.k[0], True), (got[1], plain.eng.v[0], False)):
                rows = full[unit, :, :1].cpu().expand(-1, 16, -1)
                want = ref.values(ref.pack(*ref.quantise(rows), key), key).float().to(torch.bfloat16)[:, 0]
                assert torch.equal(x[0, :, 0].cpu(), want)
    assert int(runs[0].err.item()) == 0 and int(runs[1].err.item()) == 0
