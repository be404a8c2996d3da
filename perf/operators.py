"""Cases of the paged 4-bit KV cache operators: their inputs, plain forms, 64-bit values and work.

The cache is a uint8 tensor ``pages[page][kv head][page bytes]``. A page holds ``page`` tokens in
tiles of 16; a tile is 20 D bytes: key codes (8 D), value codes (8 D), key and value parameters
(2 D each). A head vector is cut into groups of 32 dims; a group stores s and z (bf16) and one
4-bit code c per dim, standing for s c + z. With token t of the tile (r = t % 8, h = t // 8) and
dim 32 w + 16 b + 8 n + x (b, n in {0, 1}, x in 0..7), the code is nibble n (low first) of byte

    keys    (w // 2) 512 + (4 r + x // 2) 16 + h 8 + (w % 2) 4 + (x % 2) 2 + b
    values  (w // 2) 512 + (4 x + r // 2) 16 + (w % 2) 8 + h 4 + (r % 2) 2 + b

of its 8 D bytes, and the group's parameters are the 4 bytes (s, then z, little-endian) at
(2 r + h) D / 8 + 4 w of their 2 D bytes.

Operators: ``append`` (norm of each query and key head, position rotation, storing keys and
values; then ``read`` gives back what the cache holds for these tokens), ``read`` alone, and
``attend`` (each query row of a sequence over its cached keys and values).
"""

from __future__ import annotations

import math
import os
import sys

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(_ROOT, "pulsar-300m_b200"))

own = False

EPS = 1e-6


# ------------------------------------------------------------------------------------- cases
def _append(name, tokens, *, hq=16, hkv=4, d=64, page=64, rot=64, interleaved=False, norm=True, gain=False,
            decode=False):
    return {"name": name, "op": "append", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "page": page, "rot": rot,
            "interleaved": interleaved, "norm": norm, "gain": gain, "decode": decode}


def _read(name, tokens, *, hkv=4, d=64, page=64):
    return {"name": name, "op": "read", "tokens": tokens, "hkv": hkv, "d": d, "page": page}


def _attend(name, batch, q_lo, q_hi, kv_lo, kv_hi, *, window=0, hq=16, hkv=4, d=64, page=64):
    return {"name": name, "op": "attend", "batch": batch, "q_lo": q_lo, "q_hi": q_hi, "kv_lo": kv_lo, "kv_hi": kv_hi,
            "window": window, "hq": hq, "hkv": hkv, "d": d, "page": page}


def listed():
    return [
        # one sequence decodes one token: all latency
        _append("append 1 token", 1, gain=True, decode=True),
        # a decode step of 256 sequences (the throughput workload's batch)
        _append("append 256 decode tokens", 256, decode=True),
        # a long prompt prefilled in one call
        _append("append 16384 prompt tokens", 16384),
        # heads of 128 with half of each rotated in neighbouring pairs, no norm, small pages, an odd count
        _append("append 1531 interleaved d128", 1531, hq=32, hkv=8, d=128, page=16, rot=64, interleaved=True,
                norm=False),
        # a few hundred positions read back
        _read("read 777", 777, page=32),
        # a whole 32768-token sequence read back
        _read("read 32768", 32768),
        # batch-1 decode behind a 2048-token prompt (the latency workload)
        _attend("decode 1 x 2048", 1, 1, 1, 2051, 2051),
        # 256 sequences behind 512-token prompts, up to 256 tokens on, in a windowed layer
        _attend("decode 256 x 640", 256, 1, 1, 513, 767, window=1024),
        # four long contexts in a global layer
        _attend("decode 4 x 32768", 4, 1, 1, 32768, 33023),
        # ragged lengths from one token on, heads of 128, small pages
        _attend("decode 48 ragged d128", 48, 1, 1, 1, 8191, hq=32, hkv=8, d=128, page=16),
        # verify blocks of gamma + 1 = 5 rows of 64 sequences in a windowed layer
        _attend("verify 64 x 5 windowed", 64, 5, 5, 1029, 2047, window=1024),
        # a chunk of 2048 prompt rows behind 14336 cached positions
        _attend("prefill 2048 on 16384", 1, 2048, 2048, 16384, 16384),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "decode", "decode", "verify", "prefill"])
    d = rng.choice([64, 64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        decode = rng.random() < 0.4
        n = min(_log(rng, 1, 2048 if decode else 16384), 16384 * 24 * 64 // ((hq + 2 * hkv) * d))
        c = _append("", n, hq=hq, hkv=hkv, d=d, page=page, rot=rng.choice([d, d // 2, 32, 16]),
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.7, gain=rng.random() < 0.5, decode=decode)
    elif kind == "read":
        c = _read("", min(_log(rng, 1, 32768), 32768 * 4 * 64 // (hkv * d)), hkv=hkv, d=d, page=page)
    else:
        window = rng.choice([0, 0, 128, 1000, 1024])
        if kind == "prefill":
            kv = _log(rng, 200, 16384)
            q_hi = min(_log(rng, 33, 2048), kv, max(33, 120_000_000_000 // (4 * hq * d * kv)))
            batch = max(1, min(rng.randint(1, 4), 120_000_000_000 // (4 * hq * d * kv * q_hi)))
            q_lo, kv_lo, kv_hi = rng.randint(max(1, q_hi // 2), q_hi), rng.randint(max(q_hi, kv // 2), kv), kv
        else:
            kv_hi = _log(rng, 16, 33000)
            batch = max(1, min(_log(rng, 1, 256), 300_000_000 // (kv_hi * hkv * d)))
            q_lo = q_hi = 1
            if kind == "verify":
                q_hi = rng.randint(2, 8)
                q_lo = rng.randint(1, q_hi)
            kv_hi = max(kv_hi, q_hi)
            kv_lo = rng.randint(q_hi, kv_hi)
        c = _attend("", batch, q_lo, q_hi, kv_lo, kv_hi, window=window, hq=hq, hkv=hkv, d=d, page=page)
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


# ------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _keys_values(g, n, hkv, d):
    """Keys as they are after their norm and rotation (channels of unequal weight), values with offsets."""
    k = _randn(g, n, hkv, d) * torch.exp(0.3 * _randn(g, hkv, d))
    v = 0.5 * _randn(g, n, hkv, d) + 0.2 * _randn(g, hkv, d)
    return k, v


def prepare(case, seed):
    g = _gen(seed)
    d, hkv, page = case["d"], case["hkv"], case["page"]
    state = {"op": case["op"], "d": d, "page": page}
    if case["op"] in ("append", "read"):
        n = case["tokens"]
        num_pages = -(-n // page) + 3
        # a prompt fills pages in table order; decoding sequences each write somewhere in a page
        perm = torch.randperm(num_pages, generator=g, device="cuda")
        at = torch.arange(n, device="cuda")
        if case.get("decode"):
            num_pages = n + 3
            perm = torch.randperm(num_pages, generator=g, device="cuda")
            off = torch.randint(page, (n,), generator=g, device="cuda")
            slots = perm[:n] * page + off
        else:
            slots = perm[at // page] * page + at % page
        pages = torch.zeros(num_pages, hkv, 20 * d * (page // 16), dtype=torch.uint8, device="cuda")
        state |= {"pages": pages, "slots": slots}
        if case["op"] == "read":
            k, v = _keys_values(g, n, hkv, d)
            _store(pages, slots, d, *_quantise(k), *_quantise(v))
            return state
        hq, rot, max_pos = case["hq"], case["rot"], max(n, 4096) + 8
        qkv = _randn(g, n, (hq + 2 * hkv) * d).bfloat16()
        pos = torch.randint(max_pos, (n,), generator=g, device="cuda") if case["decode"] else at
        freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda").double() / rot)
        angle = torch.arange(max_pos, device="cuda").double()[:, None] * freq
        state |= {
            "q": qkv[:, :hq * d].view(n, hq, d), "k": qkv[:, hq * d:(hq + hkv) * d].view(n, hkv, d),
            "v": qkv[:, (hq + hkv) * d:].view(n, hkv, d), "positions": pos.int(),
            "cos": angle.cos().float(), "sin": angle.sin().float(), "interleaved": case["interleaved"],
            "q_norm": 1 + 0.1 * _randn(g, hq, d) if case["norm"] else None,
            "k_norm": 1 + 0.1 * _randn(g, hkv, d) if case["norm"] else None,
            "q_gain": 1 + 0.1 * torch.log((torch.arange(max_pos, device="cuda") + 1).clamp(min=1024) / 1024)
            if case["gain"] else None}
        return state
    b, hq = case["batch"], case["hq"]
    lens = torch.tensor(_spread(case["kv_lo"], case["kv_hi"], b), device="cuda")[
        torch.randperm(b, generator=g, device="cuda")]
    counts = torch.tensor(_spread(case["q_lo"], case["q_hi"], b), device="cuda")
    width = -(-case["kv_hi"] // page)
    used = -(-lens // page)
    total = int(used.sum())
    perm = torch.randperm(total + 2, generator=g, device="cuda")
    first = used.cumsum(0) - used
    col = torch.arange(width, device="cuda")
    table = torch.where(col < used[:, None], perm[(first[:, None] + col).clamp(max=total)], -1)
    pages = torch.zeros(total + 2, hkv, 20 * d * (page // 16), dtype=torch.uint8, device="cuda")
    seq = torch.repeat_interleave(torch.arange(b, device="cuda"), lens)
    at = torch.arange(len(seq), device="cuda") - (lens.cumsum(0) - lens)[seq]
    slots = table[seq, at // page] * page + at % page
    k, v = _keys_values(g, len(seq), hkv, d)
    _store(pages, slots, d, *_quantise(k), *_quantise(v))
    cu_q = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    q = (1.5 * _randn(g, int(cu_q[-1]), hq, d)).bfloat16()
    one = case["q_hi"] == 1
    state |= {"q": q, "pages": pages, "block_table": table.int(), "kv_lens": lens.int(),
              "cu_q": None if one else cu_q.int(), "max_q": case["q_hi"], "max_kv": case["kv_hi"],
              "window": case["window"]}
    return state


# -------------------------------------------------------------------------------- plain forms
def _quantise(x):
    """Codes and (s, z) of x [n, heads, d] in groups of 32 dims."""
    g = x.float().unflatten(-1, (-1, 32))
    z = g.amin(-1).bfloat16()
    s = ((g.amax(-1) - z.float()) / g.new_full((), 15.0)).bfloat16()
    s = torch.where(s.float() >= 2.0 ** -126, s, 0.0)
    c = torch.round((g - z.float()[..., None]) / torch.where(s > 0, s.float(), 1.0)[..., None]).clamp(0, 15)
    return torch.where(s[..., None] > 0, c, 0.0).flatten(-2), s, z


def _tile(pages, slots, d):
    """Byte of the start of each (slot, kv head)'s tile [n, heads], and the slot's place in it."""
    hkv, page = pages.shape[1], pages.shape[2] * 16 // (20 * d)
    heads = torch.arange(hkv, device=pages.device)
    start = ((slots // page)[:, None] * hkv + heads) * pages.shape[2] + (slots % page // 16 * 20 * d)[:, None]
    return start, slots % 16


def _places(t, d):
    """Within the tile of a token in place t [n]: its key bytes, value bytes [n, d/2] and parameters [n, d/32]."""
    w, b, x = (i.flatten() for i in torch.meshgrid(torch.arange(d // 32), torch.arange(2), torch.arange(8),
                                                   indexing="ij"))
    w, b, x = w.to(t.device), b.to(t.device), x.to(t.device)
    t = t[:, None]
    r, h = t % 8, t // 8
    k = (w // 2) * 512 + (4 * r + x // 2) * 16 + h * 8 + (w % 2) * 4 + (x % 2) * 2 + b
    v = 8 * d + (w // 2) * 512 + (4 * x + r // 2) * 16 + (w % 2) * 8 + h * 4 + (r % 2) * 2 + b
    p = (2 * r + h) * (d // 8) + 4 * torch.arange(d // 32, device=t.device)
    return k, v, p


def _bytes(c):
    """Codes [n, heads, d] as bytes [n, heads, d/2] in the order (w, b, x)."""
    c = c.to(torch.uint8).unflatten(-1, (-1, 2, 8))
    return (c[..., 0, :] + 16 * c[..., 1, :]).flatten(-2)


def _store(pages, slots, d, kc, ks, kz, vc, vs, vz):
    start, t = _tile(pages, slots, d)
    k, v, p = _places(t, d)
    flat, quads = pages.view(-1), pages.view(torch.int16).view(-1)
    flat[start[..., None] + k[:, None]] = _bytes(kc)
    flat[start[..., None] + v[:, None]] = _bytes(vc)
    at = (start[..., None] + p[:, None]) // 2
    quads[at + 8 * d], quads[at + 8 * d + 1] = ks.view(torch.int16), kz.view(torch.int16)
    quads[at + 9 * d], quads[at + 9 * d + 1] = vs.view(torch.int16), vz.view(torch.int16)


def _values(pages, d):
    """Keys and values [..., tokens, heads, d] of pages [..., heads, page bytes], in 32 bits."""
    tiles = pages.unflatten(-1, (-1, 20 * d))

    def vals(codes, dims, order, par):
        codes = codes.unflatten(-1, dims)
        codes = torch.stack([codes & 15, codes >> 4], -1)      # [..., heads, tiles, *dims, n]
        lead = codes.dim() - len(dims) - 1
        codes = codes.permute(*range(lead), *(lead + i for i in order))
        codes = codes.reshape(*codes.shape[:lead], 16, d // 32, 32)
        par = par.contiguous().view(torch.bfloat16).float().unflatten(-1, (8, 2, d // 32, 2))
        par = par.transpose(-4, -3).flatten(-4, -3)            # tokens in order (h, r)
        x = codes.float() * par[..., 0:1] + par[..., 1:2]
        return x.flatten(-2).flatten(-3, -2).transpose(-3, -2)  # [..., tokens, heads, d]

    # keys: (w/2, r, x/2, h, w%2, x%2, b, n) -> (h, r, w/2, w%2, b, n, x/2, x%2)
    k = vals(tiles[..., :8 * d], (d // 64, 8, 4, 2, 2, 2, 2), (3, 1, 0, 4, 6, 7, 2, 5), tiles[..., 16 * d:18 * d])
    # values: (w/2, x, r/2, w%2, h, r%2, b, n) -> (h, r/2, r%2, w/2, w%2, b, n, x)
    v = vals(tiles[..., 8 * d:16 * d], (d // 64, 8, 4, 2, 2, 2, 2), (4, 2, 5, 0, 3, 6, 7, 1), tiles[..., 18 * d:])
    return k, v


def _tree(s):
    """Sum over the last axis, neighbours first."""
    return s[..., 0] if s.shape[-1] == 1 else _tree(s[..., ::2] + s[..., 1::2])


def _rotate(x, c, s, interleaved):
    rot = 2 * c.shape[-1]
    c, s = c[:, None], s[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = (a * c - b * s, b * c + a * s)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, x[..., rot:]], -1)


def _norm_rotate(x, weight, st):
    x = x.float()
    if weight is not None:
        x = weight * (x * (1.0 / torch.sqrt(_tree(x * x) * (1.0 / x.shape[-1]) + EPS))[..., None])
    p = st["positions"].long()
    return _rotate(x, st["cos"][p], st["sin"][p], st["interleaved"])


def _append_plain(st):
    q = _norm_rotate(st["q"], st["q_norm"], st)
    if st["q_gain"] is not None:
        q = q * st["q_gain"][st["positions"].long()][:, None, None]
    k = _norm_rotate(st["k"], st["k_norm"], st)
    _store(st["pages"], st["slots"], st["d"], *_quantise(k), *_quantise(st["v"]))
    return q.bfloat16()


def _read_plain(st):
    d, pages = st["d"], st["pages"]
    start, t = _tile(pages, st["slots"], d)
    k, v, p = _places(t, d)
    flat, quads = pages.view(-1), pages.view(torch.int16).view(-1)
    par = (start[..., None] + p[:, None]) // 2

    def vals(at, par):
        byte = flat[start[..., None] + at[:, None]].unflatten(-1, (-1, 1, 8))
        c = torch.cat([byte & 15, byte >> 4], -2).flatten(-3).unflatten(-1, (-1, 32))
        s, z = (quads[par + i].view(torch.bfloat16).float()[..., None] for i in (0, 1))
        return (c * s + z).flatten(-2).bfloat16()

    return vals(k, par + 8 * d), vals(v, par + 9 * d)


def _attend_plain(st):
    d, q, n_kv, cu = st["d"], st["q"], st["kv_lens"].long(), st["cu_q"]
    hkv, hq, b = st["pages"].shape[1], q.shape[1], len(n_kv)
    k, v = _values(st["pages"][st["block_table"].clamp(min=0).long()], d)
    k, v = (x.flatten(1, 2).permute(0, 2, 1, 3) for x in (k, v))        # [b, hkv, keys, d]
    cu = torch.arange(b + 1, device=q.device) if cu is None else cu.long()
    n_q = cu[1:] - cu[:-1]
    j = torch.arange(st["max_q"], device=q.device)
    row = (cu[:-1, None] + j).clamp(max=len(q) - 1)                      # [b, max_q]
    pos = (n_kv - n_q)[:, None] + j
    x = q.float()[row].view(b, -1, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    s = (x @ k.transpose(-1, -2)) * d ** -0.5
    key = torch.arange(k.shape[2], device=q.device)
    seen = key <= pos[..., None]
    if st["window"]:
        seen &= key > pos[..., None] - st["window"]
    seen = seen[:, None].repeat_interleave(hq // hkv, 2)
    s = torch.where(seen, s, -math.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    y = (w @ v) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    y = y.view(b, hkv, -1, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, -1, hq, d)
    return y[j < n_q[:, None]].bfloat16()


def run(st):
    if own:
        from pulsar_b200 import paged

        if st["op"] == "attend":
            return paged.kv4_attention(st["q"], st["pages"], st["block_table"], st["kv_lens"], st["cu_q"],
                                       max_q=st["max_q"], max_kv=st["max_kv"], window=st["window"])
        if st["op"] == "append":
            q = paged.kv4_append(st["q"], st["k"], st["v"], st["pages"], st["slots"], st["positions"], st["cos"],
                                 st["sin"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS,
                                 interleaved=st["interleaved"], q_gain=st["q_gain"])
            return (q, *paged.kv4_read(st["pages"], st["slots"], st["d"]))
        return paged.kv4_read(st["pages"], st["slots"], st["d"])
    if st["op"] == "attend":
        return _attend_plain(st)
    if st["op"] == "append":
        return (_append_plain(st), *_read_plain(st))
    return _read_plain(st)


# --------------------------------------------------------------------------------------- work
def _visible(case):
    """(keys read from the cache, sum over query rows of the keys that they see)."""
    lens, counts = _spread(case["kv_lo"], case["kv_hi"], case["batch"]), _spread(case["q_lo"], case["q_hi"],
                                                                                 case["batch"])
    w = case["window"] or 1 << 40
    # the lengths are shuffled over the sequences: every row count is taken with the mean length
    mean = sum(lens) / len(lens)
    read = sum(min(n, w + sum(counts) / len(counts) - 1) for n in lens)
    seen = sum(n * min(mean - (n - 1) / 2, w) for n in counts)
    return read, seen


def work(case):
    d, hkv = case["d"], case["hkv"]
    cache = 2.5 * d / 2 * hkv                     # bytes of one token: two vectors of 5 bits a dim
    if case["op"] == "read":
        return {"bytes": case["tokens"] * (cache + 4 * hkv * d + 8), "flops": case["tokens"] * 4 * hkv * d}
    if case["op"] == "append":
        n, hq, rot = case["tokens"], case["hq"], case["rot"]
        # q, k, v in, q out; the cache written, then read back as k and v; slots, position, table rows
        b = n * (2 * (2 * hq + 2 * hkv) * d + 2 * cache + 4 * hkv * d + 16 + 4 + 4 * rot)
        return {"bytes": b, "flops": n * 10 * (hq + 2 * hkv) * d}
    read, seen = _visible(case)
    rows = sum(_spread(case["q_lo"], case["q_hi"], case["batch"]))
    return {"bytes": read * cache + rows * case["hq"] * d * 4, "flops": 4.0 * seen * case["hq"] * d}


# ------------------------------------------------------------------------------ 64-bit values
def _fetch(pages, slots, d):
    """Keys and values [n, heads, d] that the cache holds, by the byte addresses of each code."""
    raw = pages.reshape(-1).long()
    hkv, page = pages.shape[1], pages.shape[2] * 16 // (20 * d)
    s = slots.long()
    head = torch.arange(hkv, device=raw.device)
    base = ((s // page)[:, None] * hkv + head) * pages.shape[2] + ((s % page) // 16)[:, None] * (20 * d)
    base = base[..., None]
    dim = torch.arange(d, device=raw.device)
    w, b, nib, x = dim // 32, dim % 32 // 16, dim % 16 // 8, dim % 8
    r, h = (s % 8)[:, None, None], (s % 16 // 8)[:, None, None]
    at_k = base + w // 2 * 512 + 64 * r + x // 2 * 16 + 8 * h + w % 2 * 4 + x % 2 * 2 + b
    at_v = base + 8 * d + w // 2 * 512 + 64 * x + r // 2 * 16 + w % 2 * 8 + 4 * h + r % 2 * 2 + b

    def number(at):
        bits = raw[at] + 256 * raw[at + 1]
        sign, e, m = 1 - 2 * (bits >> 15), (bits >> 7) & 255, (bits & 127).double()
        return sign * torch.where(e > 0, (1 + m / 128) * torch.exp2(e.double() - 127), m * 2.0 ** -133)

    par = base + 16 * d + (2 * r + h) * (d // 8) + 4 * w
    k = ((raw[at_k] >> (4 * nib)) & 15) * number(par) + number(par + 2)
    v = ((raw[at_v] >> (4 * nib)) & 15) * number(par + 2 * d) + number(par + 2 * d + 2)
    return k, v


def _exact_stored(x):
    """The values that groups of 32 of x stand for once stored."""
    out = torch.empty_like(x)
    for i in range(0, x.shape[-1], 32):
        g = x[..., i:i + 32]
        z = g.min(-1, keepdim=True).values.to(torch.bfloat16).double()
        s = ((g.max(-1, keepdim=True).values - z) / 15).to(torch.bfloat16).double()
        c = torch.where(s > 0, torch.round((g - z) / torch.where(s > 0, s, 1.0)), 0.0).clamp(0, 15)
        out[..., i:i + 32] = s * c + z
    return out


def exact(case, seed):
    st = prepare(case, seed)
    d = case["d"]
    if case["op"] == "read":
        return _fetch(st["pages"], st["slots"], d)
    if case["op"] == "append":
        p = st["positions"].long()
        rot = case["rot"]
        c, s = st["cos"].double()[p][:, None], st["sin"].double()[p][:, None]
        got = []
        for x, weight in ((st["q"].double(), st["q_norm"]), (st["k"].double(), st["k_norm"])):
            if weight is not None:
                x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
            i = torch.arange(rot // 2, device=x.device)
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
            y = x.clone()
            y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
            got.append(y)
        if st["q_gain"] is not None:
            got[0] = got[0] * st["q_gain"].double()[p][:, None, None]
        return got[0], _exact_stored(got[1]), _exact_stored(st["v"].double())
    lens, page = st["kv_lens"].tolist(), case["page"]
    cu = list(range(len(lens) + 1)) if st["cu_q"] is None else st["cu_q"].tolist()
    out = []
    for b, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        k, v = _fetch(st["pages"], st["block_table"][b].long()[at // page] * page + at % page, d)
        q = st["q"][cu[b]:cu[b + 1]].double()
        pos = n - len(q) + torch.arange(len(q), device="cuda")
        hide = at > pos[:, None]
        if case["window"]:
            hide = hide | (at <= pos[:, None] - case["window"])
        group = case["hq"] // case["hkv"]
        y = torch.empty_like(q)
        for h in range(case["hq"]):
            s = (q[:, h] @ k[:, h // group].T / math.sqrt(d)).masked_fill(hide, -math.inf)
            y[:, h] = torch.softmax(s, -1) @ v[:, h // group]
        out.append(y)
    return torch.cat(out)
