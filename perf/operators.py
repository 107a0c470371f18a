"""The attention half of a decoder layer, as measurable cases: rotary positions, the write into a paged key-value cache and the
attention of new tokens over it.

Three paths, named by a case's ``path``:

* ``rotary``  rotation of a [tokens, heads, head_dim] tensor by its positions, or back (``inverse``, which is also the gradient).
* ``append``  keys and values of new tokens into a paged cache (bf16 or e4m3), with the rotation of q and k in the same call.
* ``attend``  attention of the last tokens of each sequence over the cache.

q, k and v of the last two are slices of one [tokens, (q heads + 2 kv heads) * head_dim] tensor, as a qkv product leaves them. Activations
are N(0, 1); queries N(0, 2), which makes some keys stand out. Pages of a sequence lie anywhere in the cache.
"""

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # a decode step of four sequences in a loop that is not captured: latency
        {"name": "rotary_decode", "path": "rotary", "tokens": 4, "heads": 10, "dim": 128, "rot": 128, "layout": "half", "dtype": "bf16", "scaled": False, "inverse": False},
        # the queries of a long prompt, far into a context stretched by the frequencies' scaling: memory bandwidth
        {"name": "rotary_prompt_scaled", "path": "rotary", "tokens": 8192, "heads": 64, "dim": 128, "rot": 128, "layout": "half", "dtype": "bf16", "scaled": True,
         "inverse": False},
        # the way back through a rotation of part of a head, in 32 bits, odd sizes
        {"name": "rotary_part_back_f32", "path": "rotary", "tokens": 1777, "heads": 20, "dim": 80, "rot": 32, "layout": "interleaved", "dtype": "f32", "scaled": False,
         "inverse": True},
        # a decode step of 64 sequences
        {"name": "append_decode_b64", "path": "append", "seqs": 64, "new": 1, "context": 600, "q_heads": 64, "kv_heads": 8, "dim": 128, "rot": 128, "layout": "half",
         "page": 64, "cache": "bf16"},
        # ragged prompts into an 8-bit cache
        {"name": "append_prompts_e4m3", "path": "append", "seqs": 8, "new": 1000, "context": 100, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 64,
         "layout": "interleaved", "page": 32, "cache": "e4m3"},
        # one short sequence: latency
        {"name": "attend_one_short", "path": "attend", "seqs": 1, "new": 1, "length": 129, "kv_heads": 8, "group": 4, "dim": 128, "page": 16, "cache": "bf16", "window": 0},
        # a serving batch with lengths of its own each
        {"name": "attend_batch", "path": "attend", "seqs": 64, "new": 1, "length": 8192, "kv_heads": 8, "group": 8, "dim": 128, "page": 64, "cache": "bf16", "window": 0},
        # two long documents: the work has to be split over the cache's length
        {"name": "attend_long", "path": "attend", "seqs": 2, "new": 1, "length": 131072, "kv_heads": 8, "group": 8, "dim": 128, "page": 64, "cache": "bf16", "window": 0},
        # the same kind of batch from an 8-bit cache
        {"name": "attend_e4m3", "path": "attend", "seqs": 32, "new": 1, "length": 16384, "kv_heads": 8, "group": 8, "dim": 128, "page": 64, "cache": "e4m3", "window": 0},
        # drafted tokens, odd head and page sizes, some sequences empty
        {"name": "attend_drafted", "path": "attend", "seqs": 24, "new": 5, "length": 4099, "kv_heads": 5, "group": 8, "dim": 96, "page": 24, "cache": "bf16", "window": 0},
        # a layer that looks back over a window only, one key head per query head
        {"name": "attend_window", "path": "attend", "seqs": 16, "new": 1, "length": 30000, "kv_heads": 16, "group": 1, "dim": 64, "page": 128, "cache": "bf16", "window": 1024},
        # many short sequences with wide heads
        {"name": "attend_many_short", "path": "attend", "seqs": 192, "new": 1, "length": 700, "kv_heads": 2, "group": 5, "dim": 256, "page": 16, "cache": "e4m3", "window": 0},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    path = rng.choice(("rotary", "append", "attend", "attend"))
    dim = 16 * rng.choice((2, 4, 4, 5, 6, 7, 8, 8, 8, 12, 16))
    rot = rng.choice((dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)))
    layout = rng.choice(("half", "interleaved"))
    if path == "rotary":
        heads = _log(rng, 1, 64)
        tokens = _log(rng, 1, max(1, min(8192, 8192 * 64 * 128 // (2 * heads * dim))))
        return {"path": path, "tokens": tokens, "heads": heads, "dim": dim, "rot": rot, "layout": layout, "dtype": rng.choice(("bf16", "bf16", "f32")),
                "scaled": rng.random() < 0.5, "inverse": rng.random() < 0.3}
    kv_heads, group = _log(rng, 1, 16), _log(rng, 1, 16)
    page = rng.choice((1, 8, 16, 16, 24, 32, 64, 64, 100, 128, 256))
    cache = rng.choice(("bf16", "e4m3"))
    if path == "append":
        new = rng.choice((1, 1, 4, _log(rng, 1, 2000)))
        seqs = _log(rng, 1, max(1, min(128, 8000 * 48 * 128 // (new * (group + 2) * kv_heads * dim))))
        return {"path": path, "seqs": seqs, "new": new, "context": _log(rng, 1, 1000), "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "rot": rot,
                "layout": layout, "page": page, "cache": cache}
    new = rng.choice((1, 1, 1, 2, rng.randint(1, 8)))
    length = _log(rng, 1, 131072)
    most = 2 * 131072 * 8 * 128 // (2 * length * kv_heads * dim * (new if new > 2 else 1))
    seqs = _log(rng, 1, max(1, min(256, most)))
    return {"path": path, "seqs": seqs, "new": new, "length": length, "kv_heads": kv_heads, "group": group, "dim": dim, "page": page, "cache": cache,
            "window": rng.choice((0, 0, _log(rng, 1, 4096)))}


# ---- states ----------------------------------------------------------------------------------------------------------------


def _frequencies(rot, scaled):
    """Inverse frequencies in 64 bits; ``scaled``: stretched 16-fold where a wavelength passes the length of the first training, blended between."""
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaled:
        turns = 8192 * inv / (2 * math.pi)  # turns over the first training's length
        keep = ((turns - 1) / (4 - 1)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / 16)
    return inv


def _magnitude(scaled):
    return 0.1 * math.log(16) + 1.0 if scaled else 1.0


def _tables(g, lengths, page, width):
    """Page tables for sequences of these lengths, and the number of pages: each sequence's pages anywhere, -1 behind them."""
    need = [(n + page - 1) // page for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g).to(torch.int32)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables.cuda(), pages


def _lengths(seqs, longest, least):
    """Lengths between an eighth of the longest and all of it, one of them the longest; with many sequences a few at the least. The same for
    every seed, so that all inputs of a case have the same shapes."""
    g = torch.Generator().manual_seed(7)
    n = (longest * (0.125 + 0.875 * torch.rand(seqs, generator=g))).ceil().long().clamp(min=least, max=longest)
    n[0] = longest
    if seqs >= 16:
        n[3::11] = least
    return n.tolist()


def _written(seqs, context, new):
    """For each sequence, how many entries its cache holds and how many tokens come to it: prompts have a quarter of the longest at least."""
    g = torch.Generator().manual_seed(7)
    before = torch.randint(0, context + 1, (seqs,), generator=g).tolist()
    share = (0.25 + 0.75 * torch.rand(seqs, generator=g)).tolist()
    return before, [new if new < 16 else max(1, int(new * f)) for f in share]


def _entries(gc, shape, kind):
    """The cache's entries: bf16, or e4m3 codes as bytes."""
    t = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gc)
    return t if kind == "bf16" else t.mul_(24).to(E4M3).view(torch.uint8)


def prepare(case, seed):
    g, gc = torch.Generator().manual_seed(seed), torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case}
    if case["path"] == "rotary":
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        t = case["tokens"]
        st["x"] = torch.empty((t, case["heads"], case["dim"]), dtype=dtype, device="cuda").normal_(generator=gc)
        far = 1000000 if case["scaled"] else 8192
        st["positions"] = (torch.arange(t) + int(torch.randint(0, far, (1,), generator=g))).cuda()
        st["inv"] = _frequencies(case["rot"], case["scaled"]).cuda()
        if own:
            from tilefish_b200 import attention as A

            st["table"] = A.RotaryTable(st["inv"], layout=case["layout"], magnitude=_magnitude(case["scaled"]))
        return st
    b, d, hk, page = case["seqs"], case["dim"], case["kv_heads"], case["page"]
    if case["path"] == "append":
        hq, new = case["q_heads"], case["new"]
        before, count = _written(b, case["context"], new)
        tables, pages = _tables(g, [p + n for p, n in zip(before, count)], page, (case["context"] + new + page - 1) // page)
        st["tables"] = tables
        st["positions"] = torch.cat([torch.arange(p, p + n) for p, n in zip(before, count)]).cuda()
        st["rows"] = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(count)]).cuda()
        t = st["positions"].numel()
        qkv = torch.empty((t, (hq + 2 * hk) * d), dtype=torch.bfloat16, device="cuda").normal_(generator=gc)
        st["q"], st["k"], st["v"] = (part.view(t, -1, d) for part in qkv.split([hq * d, hk * d, hk * d], dim=1))
        st["inv"] = _frequencies(case["rot"], False).cuda()
    else:
        hq, new = hk * case["group"], case["new"]
        lengths = _lengths(b, case["length"], 0 if new > 1 else 1)
        st["tables"], pages = _tables(g, lengths, page, (case["length"] + page - 1) // page)
        st["lengths"] = torch.tensor(lengths, dtype=torch.int32).cuda()
        st["q"] = torch.empty((b * new, hq, d), dtype=torch.bfloat16, device="cuda").normal_(generator=gc).mul_(2)
    shape = (pages, hk, page, d)
    st["kc"], st["vc"] = _entries(gc, shape, case["cache"]), _entries(gc, shape, case["cache"])
    st["scales"] = None
    if case["cache"] == "e4m3":
        st["scales"] = (0.03 + 0.02 * torch.rand(2, hk, generator=gc, device="cuda")).unbind(0)
    if own:
        from tilefish_b200 import attention as A

        st["cache"] = A.PagedCache(st["kc"], st["vc"], *(st["scales"] or ()))
        if case["path"] == "append":
            st["table"] = A.RotaryTable(st["inv"], layout=case["layout"])
    return st


# ---- the plain form ----------------------------------------------------------------------------------------------------------


def _rotated(x, positions, inv, layout, magnitude=1.0, inverse=False):
    """[tokens, heads, dim] rotated, in 32 bits, not rounded."""
    x = x.float()
    rot = 2 * inv.numel()
    angle = positions.double()[:, None] * inv
    c = (angle.cos() * magnitude).float()[:, None]
    s = (angle.sin() * (-magnitude if inverse else magnitude)).float()[:, None]
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    return torch.cat([y, x[..., rot:]], dim=-1)


def _plain_append(st):
    c = st["case"]
    q = _rotated(st["q"], st["positions"], st["inv"], c["layout"]).bfloat16()
    k = _rotated(st["k"], st["positions"], st["inv"], c["layout"])
    v = st["v"].float()
    page = st["tables"][st["rows"].long(), st["positions"] // c["page"]].long()
    slot = st["positions"] % c["page"]
    if st["scales"] is None:
        st["kc"][page, :, slot] = k.bfloat16()
        st["vc"][page, :, slot] = v.bfloat16()
        return q, st["kc"], st["vc"]
    for_cache = [(x / s[:, None]).clamp(-448, 448).to(E4M3).view(torch.uint8) for x, s in zip((k, v), st["scales"])]
    st["kc"][page, :, slot] = for_cache[0]
    st["vc"][page, :, slot] = for_cache[1]
    return q, st["kc"].view(E4M3), st["vc"].view(E4M3)


def _plain_attend(st):
    c = st["case"]
    b, n, hk, g, d = c["seqs"], c["new"], c["kv_heads"], c["group"], c["dim"]

    def gathered(entries, scale):
        e = entries[st["tables"].long().clamp(min=0)].transpose(1, 2).reshape(b, hk, -1, d)
        return e.float() if scale is None else e.view(E4M3).float() * scale[:, None, None]

    ks, vs = st["scales"] or (None, None)
    k, v = gathered(st["kc"], ks), gathered(st["vc"], vs)
    q = st["q"].float().view(b, n, hk, g, d).transpose(1, 2).reshape(b, hk, n * g, d)
    s = (q @ k.transpose(-1, -2)).view(b, hk, n, g, -1) * d**-0.5
    limit = st["lengths"].long()[:, None] - n + 1 + torch.arange(n, device="cuda")
    key = torch.arange(s.shape[-1], device="cuda")
    seen = key < limit[..., None]
    if c["window"]:
        seen = seen & (key >= limit[..., None] - c["window"])
    s = s.masked_fill(~seen[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    lse = (total.log() + top).squeeze(-1).permute(0, 2, 1, 3).reshape(b * n, hk * g)
    o = p.view(b, hk, n * g, -1) @ v / total.view(b, hk, n * g, 1).clamp(min=1e-30)
    return o.view(b, hk, n, g, d).transpose(1, 2).reshape(b * n, hk * g, d).bfloat16(), lse


def run(st):
    c = st["case"]
    if own:
        from tilefish_b200 import attention as A

        if c["path"] == "rotary":
            return A.rotary(st["x"], st["positions"], st["table"], inverse=c["inverse"])
        if c["path"] == "append":
            q = A.cache_append(st["cache"], st["k"], st["v"], st["tables"], st["positions"], rows=st["rows"], q=st["q"], rotary=st["table"])
            return (q, st["kc"], st["vc"]) if st["scales"] is None else (q, st["kc"].view(E4M3), st["vc"].view(E4M3))
        return A.paged_attention(st["q"], st["cache"], st["tables"], st["lengths"], window=c["window"], return_lse=True)
    if c["path"] == "rotary":
        return _rotated(st["x"], st["positions"], st["inv"], c["layout"], _magnitude(c["scaled"]), c["inverse"]).to(st["x"].dtype)
    return _plain_append(st) if c["path"] == "append" else _plain_attend(st)


# ---- what a pass cannot do without, and its exact result ------------------------------------------------------------------------


def work(case):
    d = case["dim"]
    if case["path"] == "rotary":
        n = case["tokens"] * case["heads"] * d
        return {"bytes": 2 * n * (2 if case["dtype"] == "bf16" else 4) + 8 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    item = 2 if case["cache"] == "bf16" else 1
    if case["path"] == "append":
        t = sum(_written(case["seqs"], case["context"], case["new"])[1])
        hq, hk = case["q_heads"], case["kv_heads"]
        return {"bytes": t * d * (4 * hq + 2 * hk * (2 + item)), "flops": 3 * t * (hq + hk) * case["rot"]}
    b, n, hk, g, longest = case["seqs"], case["new"], case["kv_heads"], case["group"], case["length"]
    lengths = _lengths(b, longest, 0 if n > 1 else 1)
    spans = sum(min(v, case["window"] + n - 1) if case["window"] else v for v in lengths)
    pairs = sum(min(max(0, v - n + 1 + i), case["window"] or v) for v in lengths for i in range(n))
    return {"bytes": 2 * spans * hk * d * item + b * n * hk * g * (4 * d + 4), "flops": 4 * pairs * hk * g * d}


def _turned(x, positions, inv, layout, magnitude=1.0, sign=1.0):
    """The rotation as a product of complex numbers, in 64 bits."""
    rot = 2 * inv.numel()
    z = x.double()[..., :rot]
    z = torch.complex(*((z[..., :rot // 2], z[..., rot // 2:]) if layout == "half" else (z[..., ::2], z[..., 1::2])))
    angle = torch.outer(positions.double(), inv) * sign
    z = z * torch.polar(torch.full_like(angle, magnitude), angle)[:, None]
    y = x.double().clone()
    if layout == "half":
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["path"] == "rotary":
        return _turned(st["x"], st["positions"], st["inv"], case["layout"], _magnitude(case["scaled"]), -1.0 if case["inverse"] else 1.0)
    quantized = case["cache"] == "e4m3"
    if case["path"] == "append":
        caches = [c.view(E4M3).double() if quantized else c.double() for c in (st["kc"], st["vc"])]
        for i, x in enumerate((_turned(st["k"], st["positions"], st["inv"], case["layout"]), st["v"].double())):
            if quantized:
                x = (x / st["scales"][i].double()[:, None]).clamp(-448, 448)
            for b in range(case["seqs"]):
                mine = st["rows"] == b
                at = st["positions"][mine]
                caches[i][st["tables"][b].long()[at // case["page"]], :, at % case["page"]] = x[mine]
        return (_turned(st["q"], st["positions"], st["inv"], case["layout"]), *caches)
    n, hk, g, d = case["new"], case["kv_heads"], case["group"], case["dim"]
    out = torch.zeros_like(st["q"], dtype=torch.float64)
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, length in enumerate(st["lengths"].tolist()):
        at = torch.arange(length, device="cuda")
        where = st["tables"][b].long()[at // case["page"]], at % case["page"]
        for h in range(hk):
            k, v = (c[where[0], h, where[1]] for c in (st["kc"], st["vc"]))
            k, v = ((x.view(E4M3).double() * st["scales"][i][h].double() if quantized else x.double()) for i, x in enumerate((k, v)))
            for i in range(n):
                stop = length - n + 1 + i
                start = max(0, stop - case["window"]) if case["window"] else 0
                if stop <= start:
                    continue
                t, heads = b * n + i, slice(h * g, (h + 1) * g)
                s = st["q"][t, heads].double() @ k[start:stop].T / math.sqrt(d)
                lse[t, heads] = torch.logsumexp(s, -1)
                out[t, heads] = torch.exp(s - lse[t, heads, None]) @ v[start:stop]
    return out, lse
