"""Measured cases of the 4-bit KV cache and of windowed attention.

Operators (public entry points in cache_eviction_b200.kernels):

  kv4_write, kv4_read     K/V rows quantised to 4 bits as they are written into
                          the paged pools, and pages read back as bf16
  kv4_decode_attn_score   one token per sequence attending to 4-bit pages, with
                          the H2O page scores of the eviction policies
  window_decode           one token per sequence attending to its first tokens
                          and to a sliding window, over bf16 pages
  window_prefill          the same mask for a prompt's chunk of queries

A case is a dict of plain values; prepare() makes its inputs on the GPU from
the seed, run() makes one pass (the plain torch form, or with `own` the
framework's call) and exact() states the result in 64 bits.

The 4-bit page: a (unit, KV head) slice of 576 bytes, 16 tokens of 64 values.
Each token has a scale s and a minimum m (bf16, bytes 512 + 4 * token: s then
m) and 64 codes c in 0..15, a value being m + c * s.  K codes: dims 16 t ..
16 t + 15 of token j are the 8 bytes at ((j / 2) * 4 + t) * 16 + (j % 2) * 8,
the even dim in a byte's low half.  V codes: byte ((j / 4 * 8 + r) * 4 + q) * 4
+ j % 4 holds dims 16 q + r (low half) and 16 q + r + 8 of token j.
"""
import math

import torch

own = False

D, P, GROUP = 64, 16, 8          # head dim, tokens per page, query heads per KV head
SLICE = P * 36                   # bytes of one (unit, KV head): 512 of codes, 64 of scales and minima
SCALE = D ** -0.5
DEV = "cuda"


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of a 64-sequence batch: each sequence's new token goes into its page, the pages come back
        dict(name="write_step", kind="write", tokens=64, heads=8, run="step"),
        # a whole prompt written into consecutive pages of a sequence and read back (odd length: the last page is partial)
        dict(name="write_prompt", kind="write", tokens=29719, heads=8, run="prompt"),
        # a page group brought back to bf16 for a prompt's next chunk
        dict(name="read_chunk", kind="read", pages=128, heads=8),
        # a 64K-token prefix brought back to bf16
        dict(name="read_prefix", kind="read", pages=4096, heads=8),
        # one short sequence: latency
        dict(name="decode4_short", kind="decode4", rows=1, shortest=517, longest=517, heads=8, mode="sum"),
        # batch 1 at ~29.7K resident tokens (the long-context single-request decode)
        dict(name="decode4_long", kind="decode4", rows=1, shortest=29719, longest=29719, heads=8, mode="sum"),
        # the ragged continuous batch: 64 sequences of 2K to 32K resident tokens, scored and unscored rows mixed
        dict(name="decode4_batch", kind="decode4", rows=64, shortest=2048, longest=32768, heads=8, mode="mixed"),
        # the same batch on one of eight GPUs: a single KV head
        dict(name="decode4_shard", kind="decode4", rows=64, shortest=2048, longest=32768, heads=1, mode="max"),
        # a sliding-window layer's decode step: 64 sequences, a 128-token window
        dict(name="step_swa", kind="step", rows=64, shortest=90, longest=4099, window=128, first=0, heads=8, page=16),
        # a streaming budget of 8,192: the first 2,048 tokens and the last 6,144 of long sequences
        dict(name="step_stream", kind="step", rows=64, shortest=4096, longest=32768, window=6144, first=2048, heads=8, page=16),
        # a prompt through a sliding-window layer
        dict(name="prompt_swa", kind="chunk", rows=2, queries=4093, prefix=0, window=128, first=0, heads=8, page=16),
        # a 2,048-query chunk behind a long prefix under a streaming budget
        dict(name="chunk_stream", kind="chunk", rows=1, queries=2048, prefix=26624, window=6144, first=2048, heads=8, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode4", "decode4", "step", "chunk"])
    heads = rng.choice([1, 2, 4, 8])
    if kind == "write":
        run = rng.choice(["step", "prompt"])
        return dict(kind=kind, tokens=_log(rng, 1, 4000 if run == "step" else 29000), heads=heads, run=run)
    if kind == "read":
        return dict(kind=kind, pages=_log(rng, 1, 4000), heads=heads)
    if kind == "decode4":
        rows, longest = _log(rng, 1, 64), _log(rng, 1, 32000)
        return dict(kind=kind, rows=rows, shortest=rng.randint(1, longest), longest=longest, heads=heads,
                    mode=rng.choice(["none", "sum", "max", "mixed"]))
    page = rng.choice([16, 16, 16, 1])
    heads = 8 if page == 1 else heads
    window, first = rng.choice([_log(rng, 1, 8000), -1]), rng.choice([0, rng.randint(1, 8), _log(rng, 1, 2048)])
    if kind == "step":
        rows, longest = _log(rng, 1, 64), _log(rng, 1, 20000)
        return dict(kind=kind, rows=rows, shortest=rng.randint(1, longest), longest=longest, window=window, first=first,
                    heads=heads, page=page)
    queries = _log(rng, 1, 2000)
    return dict(kind=kind, rows=rng.randint(1, max(1, 2000 // queries) if queries > 200 else 6), queries=queries,
                prefix=rng.choice([0, _log(rng, 1, 6000)]), window=window, first=first, heads=heads, page=page)


def _lengths(rows, lo, hi):
    """rows lengths spread over [lo, hi] evenly in their logarithm (golden-ratio steps)."""
    return [int(round(lo * (hi / lo) ** ((0.5 + i * 0.6180339887498949) % 1.0))) for i in range(rows)] if rows > 1 else [hi]


def _chunks(case):
    """(queries, prefix) of each entry: the longest first, then odd shares of it."""
    return [(max(1, case["queries"] - (i * case["queries"]) // (2 * case["rows"]) - (i % 2)),
             case["prefix"] - (i * case["prefix"]) // (case["rows"] + 1)) for i in range(case["rows"])]


def _visible(n, window, first):
    """Tokens of 0 .. n-1 that a query at n - 1 sees."""
    if window < 0 or window >= n:
        return n
    return window + min(first, n - window)


def work(case):
    G = case["heads"]
    H = GROUP * G
    kv16, kv4 = G * D * 2 * 2, G * 36 * 2              # bytes of one token's K and V
    if case["kind"] == "write":
        T = case["tokens"]
        pages = T if case["run"] == "step" else -(-(T + 5) // P)
        return dict(bytes=T * (kv16 + kv4 + 8) + pages * P * (kv4 + kv16), flops=T * G * D * 2 * 8)
    if case["kind"] == "read":
        return dict(bytes=case["pages"] * (P * (kv4 + kv16) + 4), flops=case["pages"] * P * G * D * 2 * 2)
    if case["kind"] == "decode4":
        lens = _lengths(case["rows"], case["shortest"], case["longest"])
        n, pages = sum(lens), sum(-(-x // P) for x in lens)
        scored = {"none": 0.0, "sum": 1.0, "max": 1.0, "mixed": 2.0 / 3.0}[case["mode"]]
        return dict(bytes=n * kv4 + pages * 4 + len(lens) * H * D * 2 * 2 + scored * pages * G * 8,
                    flops=n * H * D * 4)
    if case["kind"] == "step":
        lens = _lengths(case["rows"], case["shortest"], case["longest"])
        n = sum(_visible(x, case["window"], case["first"]) for x in lens)
        return dict(bytes=n * kv16 + (n // case["page"]) * 4 + len(lens) * H * D * 2 * 2, flops=n * H * D * 4)
    pairs = nq = keys = 0
    for q, pre in _chunks(case):
        pairs += sum(_visible(pre + i + 1, case["window"], case["first"]) for i in range(q))
        nq += q
        keys += q + _visible(pre + 1, case["window"], case["first"]) - 1
    return dict(bytes=nq * H * D * 2 * 2 + keys * kv16, flops=pairs * H * D * 4)


# ------------------------------------------------------------------ inputs
def _keys_like(gen, shape):
    """Cache rows as a model makes them: per-channel means and spreads, bf16."""
    G = shape[1]
    mean = torch.randn((G, 1, D), generator=gen, device=DEV) * 0.5
    spread = torch.exp(0.3 * torch.randn((G, 1, D), generator=gen, device=DEV))
    return (torch.randn(shape, generator=gen, device=DEV) * spread + mean).to(torch.bfloat16)


def _quantise(x):
    """Codes (uint8), scale and minimum (bf16) of rows x [..., 64]."""
    x = x.float()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high * 0.5 - low * 0.5) * torch.tensor(2.0 / 15.0, device=x.device)).to(torch.bfloat16)
    s = scale.float()
    code = torch.where(s > 0, torch.round((x - low) / s).clamp(0, 15), torch.zeros_like(x))
    return code.to(torch.uint8), scale, low.to(torch.bfloat16)


def _pack(x, is_key):
    """Rows x [N, G, 16, 64] bf16 as 4-bit slices [N, G, 576] uint8."""
    c, s, m = _quantise(x)
    N, G = x.shape[:2]
    if is_key:
        c = c.view(N, G, 8, 2, 4, 8, 2).permute(0, 1, 2, 4, 3, 5, 6)       # pair, block, half, byte, low/high
    else:
        c = c.view(N, G, 4, 4, 4, 2, 8).permute(0, 1, 2, 6, 4, 3, 5)       # quad, r, q, token, low/high
    c = (c[..., 0] | (c[..., 1] << 4)).reshape(N, G, 512)
    par = torch.cat((s, m), -1).contiguous().view(torch.uint8).reshape(N, G, 64)
    return torch.cat((c, par), -1)


def _pool4(gen, units, G, is_key):
    pool = torch.empty((units, G, SLICE), dtype=torch.uint8, device=DEV)
    for a in range(0, units, 8192):
        n = min(8192, units - a)
        pool[a:a + n] = _pack(_keys_like(gen, (n, G, P, D)), is_key)
    return pool


def _csr(gen, lens, page):
    """Scattered units of every sequence: (indptr, indices, tokens, pool units)."""
    counts = [-(-x // page) for x in lens]
    units = sum(counts) + 7
    order = torch.randperm(units, generator=gen, device=DEV).to(torch.int32)[:sum(counts)].contiguous()
    indptr = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
    return indptr, order, torch.tensor(lens, dtype=torch.int32, device=DEV), units


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)
    G = case["heads"]
    H = GROUP * G
    s = dict(case=case, err=torch.zeros(1, dtype=torch.int32, device=DEV))
    if case["kind"] in ("write", "read"):
        n = case["pages"] if case["kind"] == "read" else case["tokens"] if case["run"] == "step" else -(-(case["tokens"] + 5) // P)
        s["units"] = torch.randperm(n + 9, generator=gen, device=DEV).to(torch.int32)[:n].contiguous()
        s["k_pool"], s["v_pool"] = _pool4(gen, n + 9, G, True), _pool4(gen, n + 9, G, False)
        if case["kind"] == "write":
            T = case["tokens"]
            s["k"], s["v"] = (_keys_like(gen, (1, G, T, D))[0].transpose(0, 1).contiguous() for _ in range(2))
            if case["run"] == "step":
                page = torch.arange(T, device=DEV)
                slot = torch.randint(0, P, (T,), generator=gen, device=DEV)
            else:
                page, slot = (torch.arange(T, device=DEV) + 5) // P, (torch.arange(T, device=DEV) + 5) % P
            s["page"], s["slot"] = page, slot
            s["loc"] = s["units"].long()[page] * P + slot
        return s
    s["sinks"] = torch.randn(H, generator=gen, device=DEV)
    if case["kind"] == "chunk":
        parts = _chunks(case)
        lens, nq = [a + b for a, b in parts], [a for a, _ in parts]
        s["max_q"], s["max_tokens"] = max(nq), max(lens)
        s["qo_indptr"] = torch.tensor([0] + nq, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
        rows = sum(nq)
    else:
        lens = _lengths(case["rows"], case["shortest"], case["longest"])
        rows = len(lens)
        s["max_tokens"] = max(lens)
    s["q"] = (torch.randn((rows, H, D), generator=gen, device=DEV) * 1.5).to(torch.bfloat16)
    page = case.get("page", P)
    s["indptr"], s["indices"], s["tokens"], units = _csr(gen, lens, page)
    if case["kind"] == "decode4":
        s["k_pool"], s["v_pool"] = _pool4(gen, units, G, True), _pool4(gen, units, G, False)
        mode = {"none": [0], "sum": [1], "max": [2], "mixed": [1, 2, 0]}[case["mode"]]
        s["mode"] = torch.tensor([mode[i % len(mode)] for i in range(rows)], dtype=torch.int32, device=DEV)
        s["rows"] = torch.arange(rows, dtype=torch.int64, device=DEV)
        s["scores"] = torch.exp(torch.randn((G, units), generator=gen, device=DEV))
    else:
        s["k_pool"], s["v_pool"] = (_keys_like(gen, (units, G, page, D)) for _ in range(2))
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return {"write": _run_write, "read": _run_read, "decode4": _run_decode4, "step": _run_step, "chunk": _run_chunk}[s["case"]["kind"]](s)


def _codes(pool, is_key):
    """Codes (fp32) [N, G, 16, 64] and scale, minimum [N, G, 16, 1] of slices [N, G, 576]."""
    N, G = pool.shape[:2]
    b = pool[..., :512]
    c = torch.stack((b & 15, b >> 4), -1).float()
    if is_key:
        c = c.view(N, G, 8, 4, 2, 8, 2).permute(0, 1, 2, 4, 3, 5, 6)
    else:
        c = c.view(N, G, 4, 8, 4, 4, 2).permute(0, 1, 2, 5, 4, 6, 3)
    par = pool[..., 512:].contiguous().view(torch.bfloat16).view(N, G, P, 2).float()
    return c.reshape(N, G, P, D), par[..., :1], par[..., 1:]


def _values(pool, is_key):
    c, s, m = _codes(pool, is_key)
    return m + c * s


def _run_write(s):
    if own:
        from cache_eviction_b200 import kernels
        kernels.kv4_write(s["k"], s["v"], s["k_pool"], s["v_pool"], s["loc"], err=s["err"])
        return kernels.kv4_read(s["k_pool"], s["v_pool"], s["units"], err=s["err"])
    units = s["units"].long()
    out = []
    for pool, rows, is_key in ((s["k_pool"], s["k"], True), (s["v_pool"], s["v"], False)):
        x = _values(pool[units], is_key)
        code, scale, low = _quantise(rows)
        x[s["page"], :, s["slot"]] = low.float() + code.float() * scale.float()
        out.append(x.to(torch.bfloat16))
    return tuple(out)


def _run_read(s):
    if own:
        from cache_eviction_b200 import kernels
        return kernels.kv4_read(s["k_pool"], s["v_pool"], s["units"], err=s["err"])
    units = s["units"].long()
    return _values(s["k_pool"][units], True).to(torch.bfloat16), _values(s["v_pool"][units], False).to(torch.bfloat16)


def _pages(s, page):
    """Units of every sequence [B, max pages] (0 past its end) and which of them are its own."""
    most = -(-s["max_tokens"] // page)
    at = s["indptr"][:-1, None].long() + torch.arange(most, device=DEV)
    have = at < s["indptr"][1:, None]
    return torch.where(have, s["indices"].long()[at.clamp(max=s["indices"].numel() - 1)], 0), have


def _run_decode4(s):
    if own:
        from cache_eviction_b200 import kernels
        out = kernels.kv4_decode_attn_score(s["q"], s["k_pool"], s["v_pool"], s["indptr"], s["indices"], s["tokens"], SCALE,
                                            sinks=s["sinks"], mode_of_row=s["mode"], rows=s["rows"], scores=s["scores"], err=s["err"])
        return out, s["scores"]
    B, H, _ = s["q"].shape
    G = H // GROUP
    units, have = _pages(s, P)
    N = units.shape[1]
    k = _values(s["k_pool"][units.view(-1)], True).view(B, N, G, P, D)
    logit = torch.einsum("bgjd,bngpd->bgjnp", s["q"].float().view(B, G, GROUP, D), k) * SCALE
    del k
    token = torch.arange(N * P, device=DEV).view(N, P)
    logit.masked_fill_((token >= s["tokens"][:, None, None])[:, None, None], -math.inf)
    sink = s["sinks"].view(1, G, GROUP, 1, 1)
    top = torch.maximum(logit.amax((3, 4), keepdim=True), sink)
    p = torch.exp(logit - top)
    p = p / (p.sum((3, 4), keepdim=True) + torch.exp(sink - top))
    v = _values(s["v_pool"][units.view(-1)], False).view(B, N, G, P, D)
    out = torch.einsum("bgjnp,bngpd->bgjd", p, v).reshape(B, H, D).to(torch.bfloat16)
    mode = s["mode"].view(B, 1, 1)
    mass = torch.where(mode == 1, p.sum((2, 4)), torch.where(mode == 2, p.amax(2).sum(-1), 0.0))     # [B, G, N]
    # the page that the newest token starts is overwritten instead of added to
    last = units.gather(1, ((s["tokens"].long() - 1) // P)[:, None]).view(-1)
    fresh = ((s["tokens"] - 1) % P == 0) & (s["mode"] > 0)
    keep = torch.ones(s["scores"].shape[1], device=DEV)
    keep[last] = torch.where(fresh, 0.0, 1.0)
    mass = torch.where(have[:, None], mass, 0.0)
    s["scores"].mul_(keep).index_add_(1, units.view(-1), mass.transpose(0, 1).reshape(G, -1))
    return out, s["scores"]


def _attend(q, k, v, seen, sinks):
    """softmax over the visible keys and the sink: q [B, n, G, 8, D], k and v [B, T, G, D], seen [B, n, T]."""
    logit = torch.einsum("bngjd,btgd->bgjnt", q, k).mul_(SCALE)
    logit.masked_fill_(~seen[:, None, None], -math.inf)
    sink = sinks.view(1, k.shape[2], GROUP, 1, 1)
    top = torch.maximum(logit.amax(-1, keepdim=True), sink)
    p = logit.sub_(top).exp_()
    p = p.div_(p.sum(-1, keepdim=True) + torch.exp(sink - top))
    return torch.einsum("bgjnt,btgd->bngjd", p, v)


def _gathered(s, pool, units):
    B, N = units.shape
    G, page = pool.shape[1:3]
    return pool[units.view(-1)].float().view(B, N, G, page, D).transpose(2, 3).reshape(B, N * page, G, D)


def _run_step(s):
    case = s["case"]
    if own:
        from cache_eviction_b200 import kernels
        return kernels.window_decode(s["q"], s["k_pool"], s["v_pool"], s["indptr"], s["indices"], s["tokens"], SCALE, case["page"],
                                     case["window"], first=case["first"], sinks=s["sinks"], err=s["err"])
    B, H, _ = s["q"].shape
    units, _ = _pages(s, case["page"])
    t = torch.arange(units.shape[1] * case["page"], device=DEV)
    n = s["tokens"][:, None].long()
    seen = t < n
    if case["window"] >= 0:
        seen = seen & ((t >= n - case["window"]) | (t < case["first"]))
    k, v = _gathered(s, s["k_pool"], units), _gathered(s, s["v_pool"], units)
    return _attend(s["q"].float().view(B, 1, H // GROUP, GROUP, D), k, v, seen[:, None], s["sinks"]).reshape(B, H, D).to(torch.bfloat16)


def _run_chunk(s):
    case = s["case"]
    if own:
        from cache_eviction_b200 import kernels
        return kernels.window_prefill(s["q"], s["k_pool"], s["v_pool"], s["qo_indptr"], s["indptr"], s["indices"], s["tokens"], SCALE,
                                      case["page"], s["max_q"], s["max_tokens"], case["window"], first=case["first"],
                                      sinks=s["sinks"], err=s["err"])
    total, H, _ = s["q"].shape
    G = H // GROUP
    units, _ = _pages(s, case["page"])
    # every entry's queries padded to the longest chunk
    nq = (s["qo_indptr"][1:] - s["qo_indptr"][:-1]).long()
    i = torch.arange(s["max_q"], device=DEV)
    at = (s["qo_indptr"][:-1, None].long() + i).clamp(max=total - 1)
    pos = s["tokens"][:, None].long() - nq[:, None] + i
    t = torch.arange(units.shape[1] * case["page"], device=DEV)
    seen = (t <= pos[..., None]) & (t < s["tokens"][:, None, None])
    if case["window"] >= 0:
        seen = seen & ((t > pos[..., None] - case["window"]) | (t < case["first"]))
    k, v = _gathered(s, s["k_pool"], units), _gathered(s, s["v_pool"], units)
    o = _attend(s["q"].float()[at].view(len(nq), -1, G, GROUP, D), k, v, seen, s["sinks"])
    # back to the packed rows: row r belongs to the entry whose range holds it
    r = torch.arange(total, device=DEV)
    b = torch.searchsorted(s["qo_indptr"][1:].contiguous(), r.int(), right=True)
    return o[b, r - s["qo_indptr"].long()[b]].reshape(total, H, D).to(torch.bfloat16)


# ------------------------------------------------------------------ 64 bits
def _exact_rows(slices, is_key):
    """Values in 64 bits of slices [N, G, 576], nibble by nibble from the layout's formulas."""
    j = torch.arange(P, device=DEV)[:, None]
    d = torch.arange(D, device=DEV)[None, :]
    if is_key:
        byte, high = ((j // 2) * 4 + d // 16) * 16 + (j % 2) * 8 + (d % 16) // 2, d % 2 + 0 * j
    else:
        byte, high = ((j // 4 * 8 + d % 8) * 4 + d // 16) * 4 + j % 4, (d // 8) % 2 + 0 * j
    code = (slices.long()[..., byte.reshape(-1)] >> (4 * high.reshape(-1))) % 16
    par = slices[..., 512:].contiguous().view(torch.bfloat16).double().view(*slices.shape[:2], P, 2)
    return par[..., 1:] + code.double().view(*slices.shape[:2], P, D) * par[..., :1]


def _exact_softmax(q, k, v, mask, sink):
    """q [n, 8, D], k and v [T, D], mask [n, T], sink [8], all 64 bits: (p [n, 8, T], out [n, 8, D])."""
    z = (q @ k.T) * SCALE
    z = torch.where(mask[:, None], z, -math.inf)
    full = torch.cat((z, sink.view(1, -1, 1).expand(z.shape[0], -1, 1)), -1)
    p = torch.exp(z - torch.logsumexp(full, -1, keepdim=True))
    return p, p @ v


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("write", "read"):
        out = []
        for name, is_key in (("k", True), ("v", False)):
            x = _exact_rows(s[name + "_pool"][s["units"].long()], is_key)
            if kind == "write":
                r = s[name].double()
                low, high = r.min(-1, keepdim=True).values, r.max(-1, keepdim=True).values
                step = ((high - low) / 15).to(torch.bfloat16).double()
                c = torch.round((r - low) / torch.where(step > 0, step, 1.0)).clamp(0, 15)
                x[s["page"], :, s["slot"]] = low + torch.where(step > 0, c, 0.0) * step
            out.append(x)
        return tuple(out)
    G = case["heads"]
    sinks = s["sinks"].double().view(G, GROUP)
    q = s["q"].double().view(-1, G, GROUP, D)
    out = torch.zeros_like(q)
    ptr, tokens = s["indptr"].tolist(), s["tokens"].tolist()
    page = case.get("page", P)
    scores = s["scores"].double() if kind == "decode4" else None
    for b, n in enumerate(tokens):
        units = s["indices"][ptr[b]:ptr[b + 1]].long()
        if kind == "decode4":
            k, v = _exact_rows(s["k_pool"][units], True), _exact_rows(s["v_pool"][units], False)
        else:
            k, v = s["k_pool"][units].double(), s["v_pool"][units].double()
        k, v = (x.permute(1, 0, 2, 3).reshape(G, -1, D)[:, :n] for x in (k, v))
        first_row, rows = (s["qo_indptr"].tolist()[b:b + 2] if kind == "chunk" else (b, b + 1))
        for a in range(first_row, rows, 256):
            z = min(rows, a + 256)
            pos = torch.arange(n - rows + a, n - rows + z, device=DEV)[:, None]
            t = torch.arange(n, device=DEV)[None]
            mask = t <= pos
            if kind != "decode4" and case["window"] >= 0:
                mask = mask & ((pos - t < case["window"]) | (t < case["first"]))
            for g in range(G):
                p, o = _exact_softmax(q[a:z, g], k[g], v[g], mask, sinks[g])
                out[a:z, g] = o
                mode = int(s["mode"][b]) if kind == "decode4" else 0
                if mode:
                    mass = torch.zeros(len(units) * page, dtype=torch.float64, device=DEV)
                    mass[:n] = p[0].sum(0) if mode == 1 else p[0].max(0).values
                    if n % page == 1:
                        scores[g, units[-1]] = 0
                    scores[g, units] += mass.view(-1, page).sum(-1)
    out = out.reshape(-1, G * GROUP, D)
    return (out, scores) if kind == "decode4" else out
