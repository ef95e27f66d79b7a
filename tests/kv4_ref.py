"""The 4-bit page format and attention over it, stated in plain torch.

Rows are quantised in fp32 exactly as the format says (min, bf16 scale, IEEE
division, ties to even); everything computed from them is in 64 bits."""
import torch

D, P, SLICE = 64, 16, 576


def quantise(x):
    """x [..., 64] bf16 -> codes uint8 [..., 64], scale and minimum bf16 [...]."""
    bad = ~torch.isfinite(x).all(-1)
    f = torch.where(bad[..., None], torch.zeros_like(x), x).float()
    low, high = f.amin(-1), f.amax(-1)
    scale = ((high * 0.5 - low * 0.5) * torch.tensor(2.0 / 15.0)).to(torch.bfloat16)
    s = scale.float()[..., None]
    code = torch.round((f - low[..., None]) / torch.where(s > 0, s, torch.ones_like(s))).clamp(0, 15)
    code = torch.where(s > 0, code, torch.zeros_like(code)).to(torch.uint8)
    nan = torch.tensor(float("nan"), dtype=torch.bfloat16)
    low = low.to(torch.bfloat16)
    return code, torch.where(bad, nan, scale), torch.where(bad, nan, low)


def byte_of(is_key):
    """[16, 64] byte and nibble (0 low, 1 high) of every (token, dim) of a slice."""
    j, d = torch.arange(P)[:, None], torch.arange(D)[None]
    if is_key:
        return ((j // 2) * 4 + d // 16) * 16 + (j % 2) * 8 + (d % 16) // 2, d % 2 + 0 * j
    return ((j // 4) * 8 + d % 8) * 16 + (d // 16) * 4 + j % 4, (d // 8) % 2 + 0 * j


def pack(code, scale, low, is_key):
    """Slices [..., 576] of codes [..., 16, 64], scale and minimum [..., 16]."""
    byte, high = byte_of(is_key)
    out = torch.zeros((*code.shape[:-2], SLICE), dtype=torch.int64)
    out.scatter_add_(-1, byte.reshape(-1).expand(*code.shape[:-2], -1),
                     (code.long() << (4 * high)).flatten(-2))
    par = torch.stack((scale, low), -1).contiguous().view(torch.uint8).flatten(-2)
    out[..., 512:] = par.long()
    return out.to(torch.uint8)


def unpack(slices, is_key):
    """(c, s, m) in 64 bits: codes [..., 16, 64], scale and minimum [..., 16, 1]."""
    byte, high = byte_of(is_key)
    code = (slices.long()[..., byte.reshape(-1)] >> (4 * high.reshape(-1))) & 15
    par = slices[..., 512:].contiguous().view(torch.bfloat16).double().view(*slices.shape[:-1], P, 2)
    return code.double().view(*slices.shape[:-1], P, D), par[..., :1], par[..., 1:]


def values(slices, is_key):
    c, s, m = unpack(slices, is_key)
    return m + c * s


def random_pool(units, G, is_key, gen, spread=1.0):
    """Slices [units, G, 576] of random rows (a mean and a spread per channel)."""
    mean = torch.randn((1, G, 1, D), generator=gen) * 0.5
    x = ((torch.randn((units, G, P, D), generator=gen) + mean) * spread).to(torch.bfloat16)
    return pack(*quantise(x), is_key)


def attend(q, k, v, seen, sink, scale):
    """One KV head in 64 bits: q [n, 8, 64], k and v [T, 64], seen [n, T] bool,
    sink [8] or None -> p [n, 8, T], out [n, 8, 64], natural-log normaliser
    [n, 8] (rows that see nothing and have no sink: zeros and -inf)."""
    z = torch.einsum("njd,td->njt", q, k) * scale
    z = torch.where(seen[:, None], z, -torch.inf)
    full = z if sink is None else torch.cat((z, sink.view(1, -1, 1).expand(z.shape[0], -1, 1)), -1)
    lse = torch.logsumexp(full, -1) if full.shape[-1] else torch.full(z.shape[:2], -torch.inf, dtype=z.dtype)
    p = torch.where(seen[:, None], torch.exp(z - torch.where(lse.isinf(), torch.zeros_like(lse), lse)[..., None]), 0.0)
    return p, torch.einsum("njt,td->njd", p, v), lse
