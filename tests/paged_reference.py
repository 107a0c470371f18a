"""The attention operators in 64 bits, entry by entry, and how far an f32 computation of them may be off."""

import math

import torch

E4M3 = torch.float8_e4m3fn


def rotated(x, positions, inv, layout, magnitude=1.0, inverse=False):
    """(x turned, the sum of magnitudes behind each element) in 64 bits; x [tokens, heads, dim]."""
    x = x.double().cpu()
    inv = torch.as_tensor(inv, dtype=torch.float64)
    rot = 2 * inv.numel()
    i = torch.arange(rot // 2)
    i0, i1 = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    angle = positions.double().cpu()[:, None] * inv
    c, s = magnitude * angle.cos()[:, None], (-magnitude if inverse else magnitude) * angle.sin()[:, None]
    a, b = x[..., i0], x[..., i1]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    size[..., i0] = size[..., i1] = abs(magnitude) * (a.abs() + b.abs())
    return y, size


# A turned element in f32: the angle is off by half a step of an f32 in [-1, 1] half turns, pi * 2^-24 rad, and by 2^-33 turns, 0.02 * 2^-24 ...; cosine and
# sine by one step, 2^-23 (sincospif's error bound), magnitude, product and sum by half a step each. In 2^-24 of |a| + |b|: 3.2 + 2 + 1 + 1 + 1.
TURN_ERROR = 9 * 2.0**-24


def rounding(t, dtype):
    """Half a step of ``dtype`` at the values of ``t``, subnormals included."""
    tiny = {torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150, E4M3: 2.0**-10}[dtype]
    return torch.finfo(dtype).eps / 2 * t.abs() + tiny


def entries(cache_tensor, scale):
    """A cache tensor's values in 64 bits; uint8 holds e4m3 codes."""
    if cache_tensor.dtype == torch.uint8:
        t = cache_tensor.cpu().contiguous().view(E4M3).double()
        return t if scale is None else t * scale.double().cpu()[None, :, None, None]
    return cache_tensor.double().cpu()


def attention(q, k, v, tables, lengths, counts=None, scale=None, window=0, k_scale=None, v_scale=None):
    """(out, lse, bound of |out - a correct result| before its rounding, bound of lse) of the paged attention; all [tokens, heads, ...], in 64 bits."""
    k, v = entries(k, k_scale), entries(v, v_scale)
    pages, hk, page, d = k.shape
    q, tables, lengths = q.double().cpu(), tables.cpu(), lengths.cpu().tolist()
    seqs, width = tables.shape
    n_all = q.shape[0] // seqs
    g = q.shape[1] // hk
    scale = d**-0.5 if scale is None else scale
    out = torch.zeros_like(q)
    off = torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    lse_off = torch.zeros(q.shape[:2], dtype=torch.float64)
    for b in range(seqs):
        length = max(0, min(lengths[b], width * page))
        n = n_all if counts is None else max(0, min(int(counts[b]), n_all))
        for i in range(n):
            stop = length - n + 1 + i
            at = [e for e in range(max(0, stop - window) if window else 0, stop) if 0 <= int(tables[b, e // page]) < pages]
            if not at:
                continue
            e = torch.tensor(at)
            where = tables[b][e // page].long()
            for h in range(hk):
                kk, vv = k[where, h, e % page], v[where, h, e % page]
                qq = q[b * n_all + i, h * g:(h + 1) * g]
                s = qq @ kk.T * scale
                t, heads = b * n_all + i, slice(h * g, (h + 1) * g)
                lse[t, heads] = torch.logsumexp(s, -1)
                w = torch.exp(s - lse[t, heads, None])
                out[t, heads] = w @ vv
                # f32 dot products of d terms and two factors; as many additions as there are steps of at least 8 keys, and some to join them; weights
                # rounded to 11 bits at least; a weight is off by its score's error and its sum's, so twice that
                ds = (d + 6) * 2.0**-24 * abs(scale) * (qq.abs() @ kk.abs().T).amax(-1)
                steps = (len(at) / 8 + 64) * 2.0**-24
                off[t, heads] = (w @ vv.abs()) * (2.0**-11 + 2 * ds + steps)[:, None]
                lse_off[t, heads] = ds + steps + lse[t, heads].abs() * 2.0**-22
    return out, lse, off, lse_off


def check(got, want, bound, what):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= bound) & ~((got == want) | (got.isnan() & want.isnan()))
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i]} for {want[i]}, bound {torch.as_tensor(bound).expand(want.shape)[i]:.3g}")


def check_attention(out, lse, ref):
    want, want_lse, off, lse_off = ref
    check(out, want, rounding(want, torch.bfloat16) + off * (1 + 2.0**-8), "out")
    if lse is not None:
        check(lse, want_lse, lse_off, "lse")
