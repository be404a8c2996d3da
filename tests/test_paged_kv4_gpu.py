"""The paged 4-bit KV cache (pulsar_b200.paged) on the B200 against plain 64-bit evaluations.

Tolerances. A bf16 result is rounded once: relative 2^-9, taken as 2^-8 with the 32-bit work before
it. A stored value is off by half a step s / 2 plus what the rounding of s (15 s 2^-9) and of the
minimum z (|z| 2^-9) to bf16 add. Attention accumulates in 32 bits with operands good to 2^-16:
2^-12 of the largest value that a row sees, besides the rounding of the result. Above 8 units a kv
head the operands are fp16 (keys and values rounded twice, weights once, at 2^-12, and a quarter of
the weights good to 2^-13): 4 2^-12 of the largest value, and 2 2^-12 scale sum |q k| in a score, so
twice that in a weight over their sum."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    from pulsar_b200 import paged
    return paged


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# ---------------------------------------------------------------- plain evaluations, 64 bits, CPU
def held(pages, head_dim):
    """Keys and values [num_pages, page_size, heads, D] (double) that a cache holds, from its bytes."""
    raw = pages.cpu()
    tiles = raw.unflatten(-1, (-1, 20 * head_dim))            # [pages, heads, tiles, bytes]
    out = []
    for is_v in (False, True):
        codes, par = torch.zeros(*tiles.shape[:3], 16, head_dim), []
        p = tiles[..., (18 if is_v else 16) * head_dim:][..., :2 * head_dim].contiguous().view(torch.bfloat16).double()
        p = p.unflatten(-1, (8, 2, head_dim // 32, 2))        # token = (t % 8, t // 8)
        for t in range(16):
            r, h = t % 8, t // 8
            par.append(p[..., r, h, :, :])
            for w in range(head_dim // 32):
                for b in range(2):
                    for x in range(8):
                        if is_v:
                            at = 8 * head_dim + w // 2 * 512 + (4 * x + r // 2) * 16 + w % 2 * 8 + h * 4 + r % 2 * 2 + b
                        else:
                            at = w // 2 * 512 + (4 * r + x // 2) * 16 + h * 8 + w % 2 * 4 + x % 2 * 2 + b
                        byte = tiles[..., at]
                        codes[..., t, 32 * w + 16 * b + x] = (byte & 15).float()
                        codes[..., t, 32 * w + 16 * b + 8 + x] = (byte >> 4).float()
        par = torch.stack(par, -3)                            # [pages, heads, tiles, 16, groups, 2]
        val = codes.double().unflatten(-1, (-1, 32)) * par[..., 0:1] + par[..., 1:2]
        out.append(val.flatten(-2).flatten(2, 3).transpose(1, 2))
    return out


def plain_append(x, weight, eps, cos, sin, pos, interleaved):
    x = x.cpu().double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.cpu().double()
    if cos is None:
        return x
    c, s = cos.cpu().double()[pos.cpu().long()][:, None], sin.cpu().double()[pos.cpu().long()][:, None]
    half = c.shape[-1]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def plain_attention(q, k, v, table, lens, cu, scale, window):
    """k, v: held() of the cache; every row in 64 bits."""
    q = q.cpu().double()
    group, page = q.shape[1] // k.shape[2], k.shape[1]
    out = torch.zeros_like(q)
    top = torch.zeros(q.shape[0], q.shape[1], 1, dtype=torch.double)   # the largest value a row sees
    amp = torch.zeros_like(top)                                        # the largest scale sum |q k|
    for b, n in enumerate(lens):
        rows = range(cu[b], cu[b + 1])
        for j, row in enumerate(rows):
            pos = n - len(rows) + j
            keys = [i for i in range(max(0, pos - window + 1) if window else 0, pos + 1)
                    if 0 <= table[b][i // page] < k.shape[0]]
            if not keys:
                continue
            at = torch.tensor(keys)
            pg = torch.tensor([table[b][i // page] for i in keys])
            kk, vv = k[pg, at % page], v[pg, at % page]               # [keys, heads, D]
            for h in range(q.shape[1]):
                p = torch.softmax(kk[:, h // group] @ q[row, h] * scale, 0)
                out[row, h] = p @ vv[:, h // group]
                top[row, h] = vv[:, h // group].abs().max()
                amp[row, h] = (kk[:, h // group].abs() @ q[row, h].abs()).max() * scale
    return out, top, amp


def assert_attention(got, ref, top, amp, many=False):
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got.float()).all()
    rel = 4 * 2.0 ** -12 + 4 * 2.0 ** -12 * amp if many else 2.0 ** -12
    worst = (err - (2.0 ** -8 * ref.abs() + rel * top)).max().item()
    assert worst <= 0, f"off by {err.max().item():.3e}, {worst:.3e} over the bound"


# ------------------------------------------------------------------------------- append and read
@pytest.mark.parametrize("n,hq,hkv,d,page,rot,interleaved,norm,gain", [
    (1, 16, 4, 64, 64, 64, False, True, True),
    (37, 16, 4, 64, 64, 64, False, True, False),
    (50, 3, 1, 64, 16, 32, False, False, False),
    (33, 6, 2, 64, 32, 16, False, True, True),
    (21, 4, 4, 64, 128, 64, True, True, False),
    (40, 8, 2, 128, 16, 64, True, False, True),
    (19, 4, 2, 128, 64, 128, False, True, False),
    (18, 4, 2, 128, 64, 6, True, True, False),
    (17, 5, 5, 64, 64, 0, False, False, False),
])
def test_append_and_read(paged, n, hq, hkv, d, page, rot, interleaved, norm, gain):
    qkv = _randn(n, n, (hq + 2 * hkv) * d).cuda().bfloat16()
    q, k, v = (qkv[:, a * d:b * d].view(n, -1, d) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    pages = paged.kv4_pages(n // page + 3, hkv, d, page)
    slots = torch.randperm(pages.shape[0] * page, generator=torch.Generator().manual_seed(3))[:n].cuda()
    pos = torch.randint(500, (n,), generator=torch.Generator().manual_seed(4)).int().cuda()
    cos, sin = paged.rope_tables(500, rot) if rot else (None, None)
    qw, kw = (1 + 0.1 * _randn(5, hq, d).cuda(), 1 + 0.1 * _randn(6, hkv, d).cuda()) if norm else (None, None)
    qg = (1 + 0.2 * torch.rand(500, generator=torch.Generator().manual_seed(7))).cuda() if gain else None
    out = paged.kv4_append(q, k, v, pages, slots, pos, cos, sin, q_norm=qw, k_norm=kw, eps=1e-5,
                           interleaved=interleaved, q_gain=qg)
    ref = plain_append(q, qw, 1e-5, cos, sin, pos, interleaved)
    if gain:
        ref = ref * qg.cpu().double()[pos.cpu().long()][:, None, None]
    assert out.dtype == torch.bfloat16 and out.shape == (n, hq, d)
    assert ((out.cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -20).all()

    heldk, heldv = held(pages, d)
    sl = slots.cpu()
    rk, rv = paged.kv4_read(pages, slots, d)
    for name, x, y, back in (("k", plain_append(k, kw, 1e-5, cos, sin, pos, interleaved), heldk, rk),
                             ("v", v.cpu().double(), heldv, rv)):
        y = y[sl // page, sl % page]
        g = x.unflatten(-1, (-1, 32))
        mn, mx = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        step = (mx - mn) / 15
        bound = step * (0.5 + 15 * 2.0 ** -8) + mn.abs() * 2.0 ** -8 + 2.0 ** -20
        err = (y.unflatten(-1, (-1, 32)) - g).abs()
        assert (err <= bound).all(), f"{name}: {(err - bound).max().item():.3e} over the bound"
        assert torch.equal(back.cpu(), y.bfloat16()), f"{name}: read differs from what the bytes say"


def test_append_writes_nothing_else(paged):
    """Tokens without a slot, or with a position outside the tables, are not stored; other bytes stay."""
    n, d = 9, 64
    q, k, v = (_randn(i, n, 2, d).cuda().bfloat16() for i in range(3))
    pages = paged.kv4_pages(3, 2, d, 16).fill_(0xAB)
    before = pages.clone()
    slots = torch.tensor([0, -1, 48, 1 << 40, 17, 33, 47, -(1 << 40), 5]).cuda()
    pos = torch.tensor([0, 1, 2, 3, -1, 8, 7, 1, 2]).int().cuda()
    cos, sin = paged.rope_tables(8)
    out = paged.kv4_append(q, k, v, pages, slots, pos, cos, sin)
    stored = [0, 6, 8]           # tokens 4 and 5 have no table row, the others no slot
    assert (out[[4, 5]] == 0).all() and (out[[0, 1, 2, 3, 6, 7, 8]] != 0).any(-1).all()
    only = before.clone()
    paged.kv4_append(None, k[stored], v[stored], only, slots[stored], pos[stored], cos, sin)
    assert torch.equal(only, pages)
    changed = (pages != before).sum().item()
    assert 0 < changed <= 3 * 2 * 80
    zk, zv = paged.kv4_read(pages, slots[[1, 2, 3, 7]], d)
    assert (zk == 0).all() and (zv == 0).all()


def test_stored_codes_follow_the_definition(paged):
    """Values need no arithmetic before they are quantised: codes and parameters are exact, ties included."""
    d, n = 64, 64
    v = (_randn(1, n, 1, d) * torch.logspace(-30, 30, n)[:, None, None]).bfloat16()
    v[3] = 0.0
    v[4] = 2.5
    v[5, 0, :32] = torch.arange(32) / 2          # ties
    v[6, 0, 7] = float("nan")
    v[7, 0, 40] = float("inf")
    v[8, 0, 0] = -float("inf")
    v[9, 0, :32] = torch.linspace(-3e38, 3e38, 32)
    pages = paged.kv4_pages(4, 1, d, 16)
    slots = torch.arange(n).cuda()
    paged.kv4_append(None, v.cuda(), v.cuda(), pages, slots)
    hk, hv = (x.flatten(0, 1) for x in held(pages, d))
    g = v.double().unflatten(-1, (-1, 32))
    z = g.amin(-1, keepdim=True).bfloat16().double()
    s = ((g.amax(-1, keepdim=True).float() - z.float()) / 15).bfloat16().double()
    c = torch.where(s > 0, torch.round((g - z) / torch.where(s > 0, s, 1.0)), 0.0).clamp(0, 15)
    ref = torch.where(torch.isfinite(g).all(-1, keepdim=True), s * c + z, math.nan).flatten(-2)
    ref[9, 0, :32] = math.nan                    # its span is no 32-bit number
    assert torch.equal(torch.isnan(ref), torch.isnan(hv))
    assert torch.equal(ref.nan_to_num(7.0), hv.nan_to_num(7.0)) and torch.equal(hk.nan_to_num(7.0), hv.nan_to_num(7.0))


@pytest.mark.parametrize("n,d,rot,interleaved", [(300, 64, 64, False), (2000, 64, 32, False), (300, 128, 128, True),
                                                 (1500, 128, 64, False), (1200, 64, 64, True)])
def test_queries_and_codes_match_plain_32_bits(paged, n, d, rot, interleaved):
    """Every operation is rounded on its own and sums run neighbours first, so 32-bit torch operations in
    that order give the same bits (a contracted product and sum would not)."""
    hq, hkv = 4, 2
    q, k = _randn(1, n, hq, d).bfloat16().cuda(), _randn(2, n, hkv, d).bfloat16().cuda()
    qw, kw = 1 + 0.1 * _randn(3, hq, d).cuda(), 1 + 0.1 * _randn(4, hkv, d).cuda()
    cos, sin = paged.rope_tables(n, rot)
    pos = torch.randperm(n, generator=torch.Generator().manual_seed(1)).int().cuda()
    gain = 1 + torch.rand(n, generator=torch.Generator().manual_seed(2)).cuda()
    pages = paged.kv4_pages(n // 64 + 1, hkv, d)
    slots = torch.arange(n).cuda()
    out = paged.kv4_append(q, k, k, pages, slots, pos, cos, sin, q_norm=qw, k_norm=kw, interleaved=interleaved,
                           q_gain=gain)

    def plain(x, w):
        x = x.float()
        s = x * x
        while s.shape[-1] > 1:
            s = s[..., ::2] + s[..., 1::2]
        x = w * (x * (1.0 / torch.sqrt(s * (1.0 / d) + 1e-6)))
        c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
        a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
        y = x.clone()
        if interleaved:
            y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
        else:
            y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
        return y

    assert torch.equal(out, (plain(q, qw) * gain[pos.long()][:, None, None]).bfloat16())
    g = plain(k, kw).unflatten(-1, (-1, 32))
    z = g.amin(-1, keepdim=True).bfloat16().float()
    s = ((g.amax(-1, keepdim=True) - z) / g.new_full((), 15.0)).bfloat16().float()
    c = torch.round((g - z) / s).clamp(0, 15)
    assert torch.equal(paged.kv4_read(pages, slots, d)[0], (c * s + z).flatten(-2).bfloat16())


@pytest.mark.parametrize("d,page,start,shuffle", [(64, 64, 0, False), (64, 16, 5, False), (128, 32, 0, False),
                                                  (128, 64, 15, False), (64, 64, 0, True)])
def test_many_tokens_match_few(paged, d, page, start, shuffle):
    """A call of many tokens (whole tiles, a first tile begun elsewhere, scattered slots, some without a
    slot) stores and reads the same bits as calls of few."""
    n, hq, hkv = 2100, 6, 2
    q, k, v = (_randn(i, n, h, d).bfloat16().cuda() for i, h in ((1, hq), (2, hkv), (3, hkv)))
    pages = paged.kv4_pages(n // page + 3, hkv, d, page)
    order = torch.randperm(pages.shape[0], generator=torch.Generator().manual_seed(1))
    at = torch.arange(n) + start
    if shuffle:
        at = at[torch.randperm(n, generator=torch.Generator().manual_seed(2))]
    slots = (order[at // page] * page + at % page).cuda()
    slots[[7, 600, 601, 2050]] = torch.tensor([-1, 1 << 40, -7, pages.shape[0] * page]).cuda()
    pos = torch.arange(n).int().cuda()
    pos[[40, 1111]] = torch.tensor([-1, n]).int().cuda()
    cos, sin = paged.rope_tables(n, d // 2)
    w = 1 + 0.1 * _randn(5, hkv, d).cuda()
    few = pages.clone()
    out = paged.kv4_append(q, k, v, pages, slots, pos, cos, sin, k_norm=w)
    parts = []
    for a in range(0, n, 700):
        b = slice(a, a + 700)
        parts.append(paged.kv4_append(q[b], k[b], v[b], few, slots[b], pos[b], cos, sin, k_norm=w))
    assert torch.equal(out, torch.cat(parts)) and torch.equal(pages, few)
    many = paged.kv4_read(pages, slots, d)
    few = [paged.kv4_read(pages, slots[a:a + 700], d) for a in range(0, n, 700)]
    for i in (0, 1):
        assert torch.equal(many[i], torch.cat([x[i] for x in few]))
    assert (out[[40, 1111]] == 0).all() and (many[0][[7, 600, 601, 2050]] == 0).all()


@pytest.mark.parametrize("n,d,rot", [(70, 64, 48), (70, 128, 96), (40, 128, 112), (40, 128, 32), (9, 64, 16)])
def test_partial_rotation_matches_plain_32_bits(paged, n, d, rot):
    """Pairs (i, i + rot / 2) of the first dims: a partner's dims lie anywhere in the vector."""
    q = _randn(1, n, 5, d).bfloat16().cuda()
    k = _randn(2, n, 1, d).bfloat16().cuda()
    cos, sin = paged.rope_tables(n, rot)
    pos = torch.randperm(n, generator=torch.Generator().manual_seed(1)).int().cuda()
    pages = paged.kv4_pages(n // 16 + 1, 1, d, 16)
    out = paged.kv4_append(q, k, k, pages, torch.arange(n).cuda(), pos, cos, sin)
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    y = q.float()
    a, b = y[..., :rot // 2].clone(), y[..., rot // 2:rot].clone()
    y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    assert torch.equal(out, y.bfloat16())


@pytest.mark.parametrize("n,d,rot,interleaved", [(2501, 64, 64, False), (6501, 64, 0, False), (2003, 128, 128, False),
                                                 (2100, 128, 64, False), (2100, 64, 48, False), (2100, 64, 64, True),
                                                 (2100, 128, 30, True)])
def test_several_heads_a_warp(paged, n, d, rot, interleaved):
    """Head counts that fill a warp's share of heads or leave a part of one: the same bits as in calls of
    few tokens."""
    hq, hkv, page = 41, 9, 64
    q, k, v = (_randn(i, n, h, d).bfloat16().cuda() for i, h in ((1, hq), (2, hkv), (3, hkv)))
    pages = paged.kv4_pages(n // page + 1, hkv, d, page)
    slots, pos = torch.arange(n).flip(0).cuda(), torch.arange(n).int().cuda()
    cos, sin = paged.rope_tables(n, rot) if rot else (None, None)
    qw, kw = 1 + 0.1 * _randn(4, hq, d).cuda(), 1 + 0.1 * _randn(5, hkv, d).cuda()
    few, parts = pages.clone(), []
    out = paged.kv4_append(q, k, v, pages, slots, pos, cos, sin, q_norm=qw, k_norm=kw, interleaved=interleaved)
    for a in range(0, n, 300):
        b = slice(a, a + 300)
        parts.append(paged.kv4_append(q[b], k[b], v[b], few, slots[b], pos[b], cos, sin, q_norm=qw, k_norm=kw,
                                       interleaved=interleaved))
    assert torch.equal(out, torch.cat(parts)) and torch.equal(pages, few)
    many = paged.kv4_read(pages, slots, d)
    few = [paged.kv4_read(pages, slots[a:a + 300], d) for a in range(0, n, 300)]
    for i in (0, 1):
        assert torch.equal(many[i], torch.cat([x[i] for x in few]))


def test_append_empty_and_no_queries(paged):
    pages = paged.kv4_pages(2, 2)
    e = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert paged.kv4_append(e, e, e, pages, none).shape == (0, 2, 64)
    assert paged.kv4_append(None, e, e, pages, none) is None
    assert paged.kv4_read(pages, none)[0].shape == (0, 2, 64)


# ------------------------------------------------------------------------------------- attention
def _filled(paged, lens, hkv, d, page, seed=0, spare=1, fill=0xFF):
    """A cache with the given sequences on shuffled pages; unused places hold bytes `fill` (0xFF: NaN)."""
    used = [-(-n // page) for n in lens]
    total = sum(used) + spare
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(1, max(used))
    table, slots = [], []
    for n, u in zip(lens, used):
        mine = [perm.pop() for _ in range(u)]
        table.append(mine + [-1] * (width - u))
        slots += [mine[i // page] * page + i % page for i in range(n)]
    pages = paged.kv4_pages(total, hkv, d, page).fill_(fill)
    if slots:
        k = _randn(seed + 1, len(slots), hkv, d) * 1.3
        v = _randn(seed + 2, len(slots), hkv, d) + 0.3 * _randn(seed + 3, hkv, d)
        paged.kv4_append(None, k.cuda().bfloat16(), v.cuda().bfloat16(), pages, torch.tensor(slots).cuda())
    return pages, table


def _attend(paged, lens, counts, hq, hkv, d, page, window=0, scale=None, seed=0, one=False, max_q=None, **kw):
    pages, table = _filled(paged, lens, hkv, d, page, seed)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    q = (1.5 * _randn(seed + 9, cu[-1], hq, d)).bfloat16().cuda()
    t = torch.tensor(table, dtype=torch.int32).cuda()
    got = paged.kv4_attention(q, pages, t, torch.tensor(lens, dtype=torch.int32).cuda(),
                              None if one else torch.tensor(cu, dtype=torch.int32).cuda(),
                              max_q=max_q or max(1, max(counts)), window=window, scale=scale, **kw)
    k, v = held(pages, d)
    ref, top, amp = plain_attention(q, k, v, table, lens, cu, d ** -0.5 if scale is None else scale, window)
    assert_attention(got, ref, top, amp, (max_q or max(counts)) * (hq // hkv) > 8)
    return got


@pytest.mark.parametrize("hq,hkv,d,page", [(16, 4, 64, 64), (4, 1, 64, 16), (3, 3, 64, 32), (14, 2, 64, 128),
                                           (8, 1, 64, 64), (20, 1, 64, 16), (8, 2, 128, 16), (7, 1, 128, 64),
                                           (24, 1, 128, 32)])
def test_decode_lengths(paged, hq, hkv, d, page):
    """One row a sequence: from no key over one, tile and page edges to a few hundred."""
    lens = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 300]
    got = _attend(paged, lens, [1] * len(lens), hq, hkv, d, page, one=True)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("window", [1, 5, 16, 100, 1000])
def test_decode_window(paged, window):
    lens = [1, 5, 16, 17, 100, 101, 260]
    _attend(paged, lens, [1] * len(lens), 8, 2, 64, 32, window=window, one=True)


@pytest.mark.parametrize("hq,hkv,d,window", [(16, 4, 64, 0), (16, 4, 64, 20), (6, 2, 128, 0), (6, 2, 128, 33),
                                             (7, 7, 64, 0), (16, 1, 64, 40)])
def test_verify_rows(paged, hq, hkv, d, window):
    """A few rows a sequence, none of them for some, more rows than keys for others."""
    _attend(paged, [5, 40, 70, 3, 129, 64, 0, 9], [5, 1, 8, 5, 3, 0, 2, 7], hq, hkv, d, 16, window=window)


@pytest.mark.parametrize("hq,hkv,d,page,window", [(4, 1, 64, 64, 0), (4, 1, 64, 16, 70), (8, 4, 128, 32, 0),
                                                  (3, 3, 64, 128, 50), (7, 1, 128, 16, 33), (8, 2, 64, 32, 1)])
def test_prompt_rows(paged, hq, hkv, d, page, window):
    """Whole prompts and chunks behind cached keys: more units than one tile holds, few, none."""
    _attend(paged, [100, 75, 150, 33, 20], [100, 40, 65, 1, 0], hq, hkv, d, page, window=window)


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_rows_longer_than_their_keys(paged, d):
    """Rows before the first key see none of them."""
    got = _attend(paged, [50, 0, 129], [90, 33, 140], 4, 2, d, 16)
    assert (got[:40] == 0).all() and (got[90:123] == 0).all() and (got[123:134] == 0).all()


@pytest.mark.parametrize("d,window", [(64, 0), (128, 0), (64, 300)])
def test_prompt_rows_behind_many_keys(paged, d, window):
    """A few dozen rows on a long context: the keys are split over CTAs."""
    _attend(paged, [1500, 700], [20, 9], 4, 2, d, 64, window=window)
    _attend(paged, [2600], [40], 2, 2, d, 16, window=window)


def test_prompt_values_of_any_size(paged):
    """Keys and values far from 1, and of unequal size along the sequence, keep their precision."""
    lens, page, d = [400], 64, 64
    for kx, vx in ((2.0 ** -20, 2.0 ** 25), (2.0 ** 12, 2.0 ** -30)):
        pages, table = _filled(paged, lens, 1, d, page)
        k = _randn(1, 400, 1, d) * kx
        v = _randn(2, 400, 1, d) * vx * torch.linspace(-3, 3, 400).exp2()[:, None, None]
        slots = torch.tensor([table[0][i // page] * page + i % page for i in range(400)])
        paged.kv4_append(None, k.cuda().bfloat16(), v.cuda().bfloat16(), pages, slots.cuda())
        q = _randn(3, 60, 2, d).bfloat16().cuda()
        got = paged.kv4_attention(q, pages, torch.tensor(table, dtype=torch.int32).cuda(),
                                  torch.tensor(lens, dtype=torch.int32).cuda(),
                                  torch.tensor([0, 60], dtype=torch.int32).cuda(), max_q=60, scale=0.2 / kx)
        hk, hv = held(pages, d)
        assert_attention(got, *plain_attention(q, hk, hv, table, lens, [0, 60], 0.2 / kx, 0), many=True)


# The kernel for many rows is chosen where it costs less, so small calls reach it through a bound of rows
# that they do not fill.
@pytest.mark.parametrize("hq,hkv,d,page,window", [(16, 4, 64, 64, 0), (4, 1, 64, 16, 50), (3, 3, 64, 32, 0), (7, 1, 64, 128, 0),
                                                  (8, 2, 128, 16, 0), (6, 1, 128, 64, 40)])
def test_rows_below_a_large_bound(paged, hq, hkv, d, page, window):
    _attend(paged, [100, 75, 150, 33, 20], [100, 40, 65, 1, 0], hq, hkv, d, page, window=window, max_q=8192)


@pytest.mark.parametrize("d", [64, 128])
def test_rows_below_a_large_bound_longer_than_their_keys(paged, d):
    got = _attend(paged, [50, 0, 129], [90, 33, 140], 4, 2, d, 16, max_q=8192)
    assert (got[:40] == 0).all() and (got[90:123] == 0).all() and (got[123:134] == 0).all()


@pytest.mark.parametrize("d,window", [(64, 0), (128, 0), (64, 300)])
def test_rows_below_a_large_bound_behind_many_keys(paged, d, window):
    _attend(paged, [1500, 700], [20, 9], 4, 2, d, 64, window=window, max_q=4096)
    _attend(paged, [2600], [40], 2, 2, d, 16, window=window, max_q=4096)


@pytest.mark.parametrize("window", [0, 3000])
def test_chunk_behind_several_thousand_keys(paged, window):
    """Enough keys that the kernel for many rows takes few of them, in many splits."""
    _attend(paged, [4300], [17], 8, 2, 64, 64, window=window)


def test_values_of_any_size_below_a_large_bound(paged):
    lens, page, d = [300], 64, 128
    for kx, vx in ((2.0 ** -20, 2.0 ** 25), (2.0 ** 12, 2.0 ** -30)):
        pages, table = _filled(paged, lens, 1, d, page)
        k, v = _randn(1, 300, 1, d) * kx, _randn(2, 300, 1, d) * vx * torch.linspace(-3, 3, 300).exp2()[:, None, None]
        slots = torch.tensor([table[0][i // page] * page + i % page for i in range(300)])
        paged.kv4_append(None, k.cuda().bfloat16(), v.cuda().bfloat16(), pages, slots.cuda())
        q = _randn(3, 60, 2, d).bfloat16().cuda()
        got = paged.kv4_attention(q, pages, torch.tensor(table, dtype=torch.int32).cuda(),
                                  torch.tensor(lens, dtype=torch.int32).cuda(),
                                  torch.tensor([0, 60], dtype=torch.int32).cuda(), max_q=8192, scale=0.2 / kx)
        hk, hv = held(pages, d)
        assert_attention(got, *plain_attention(q, hk, hv, table, lens, [0, 60], 0.2 / kx, 0), many=True)


def test_nan_stays_where_it_is_seen_below_a_large_bound(paged):
    lens, page, rows = [40], 16, 20
    pages, table = _filled(paged, lens, 1, 64, page)
    at = torch.tensor([table[0][2] * page + 5]).cuda()          # key 37
    bad = torch.full((1, 1, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    paged.kv4_append(None, bad, bad, pages, at)
    t, n = torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    q, cu = _randn(5, rows, 4, 64).bfloat16().cuda(), torch.tensor([0, rows], dtype=torch.int32).cuda()
    got = paged.kv4_attention(q, pages, t, n, cu, max_q=8192)   # rows at positions 20 .. 39
    assert torch.isfinite(got[:17].float()).all() and torch.isnan(got[17:].float()).all()
    good, half = torch.ones_like(bad), torch.ones_like(bad)
    half[..., 40] = float("inf")
    paged.kv4_append(None, good, half, pages, at)
    for window in (0, 2):
        got = paged.kv4_attention(q, pages, t, n, cu, max_q=8192, window=window).float()
        sees = torch.zeros(rows, dtype=torch.bool)
        sees[rows - 3:rows - 1 if window else rows] = True
        assert torch.isfinite(got[..., :32]).all() and torch.isfinite(got[~sees]).all()
        assert torch.isnan(got[sees][..., 32:]).all()


def test_peaked_scores_and_missing_pages_below_a_large_bound(paged):
    _attend(paged, [200, 90], [70, 20], 4, 1, 64, 64, scale=4.0, max_q=8192)
    lens, page = [200, 90], 32
    pages, table = _filled(paged, lens, 2, 64, page)
    table[0][1], table[0][4], table[1][0] = -1, 1 << 20, pages.shape[0]
    q = _randn(4, 2, 8, 64).bfloat16().cuda()
    got = paged.kv4_attention(q, pages, torch.tensor(table, dtype=torch.int32).cuda(),
                              torch.tensor(lens, dtype=torch.int32).cuda(),
                              torch.tensor([0, 1, 2], dtype=torch.int32).cuda(), max_q=8192)
    k, v = held(pages, 64)
    assert_attention(got, *plain_attention(q, k, v, table, lens, [0, 1, 2], 0.125, 0), many=True)


@pytest.mark.parametrize("hq,d", [(4, 64), (7, 128)])
@pytest.mark.parametrize("kx,vx", [(2.0 ** -20, 2.0 ** 25), (2.0 ** 12, 2.0 ** -30), (1.0, 2.0 ** 32)])
def test_decode_values_of_any_size(paged, hq, d, kx, vx):
    lens, page = [400], 64
    pages, table = _filled(paged, lens, 1, d, page)
    k = _randn(1, 400, 1, d) * kx
    v = _randn(2, 400, 1, d) * vx * torch.linspace(-3, 3, 400).exp2()[:, None, None]
    slots = torch.tensor([table[0][i // page] * page + i % page for i in range(400)])
    paged.kv4_append(None, k.cuda().bfloat16(), v.cuda().bfloat16(), pages, slots.cuda())
    q = _randn(3, 1, hq, d).bfloat16().cuda()
    got = paged.kv4_attention(q, pages, torch.tensor(table, dtype=torch.int32).cuda(),
                              torch.tensor(lens, dtype=torch.int32).cuda(), scale=0.2 / kx)
    hk, hv = held(pages, d)
    assert_attention(got, *plain_attention(q, hk, hv, table, lens, [0, 1], 0.2 / kx, 0))


@pytest.mark.parametrize("d,window,max_kv", [(64, 0, None), (64, 0, 2500), (128, 0, None), (64, 900, None), (64, 0, 64)])
def test_decode_splits(paged, d, window, max_kv):
    """Long sequences among short ones: the keys are split over CTAs (also when max_kv is short of the truth)."""
    lens = [2500, 1, 1300, 0, 2049]
    _attend(paged, lens, [1] * len(lens), 4, 1, d, 64, window=window, one=True, max_kv=max_kv)
    _attend(paged, lens, [3, 1, 2, 1, 0], 4, 1, d, 64, window=window, max_kv=max_kv)


@pytest.mark.parametrize("hq,hkv,d,rows,window", [(4, 1, 64, 1, 0), (16, 4, 64, 1, 700), (8, 1, 128, 1, 0), (4, 1, 64, 3, 0),
                                                  (4, 2, 128, 5, 600)])
def test_decode_few_splits(paged, hq, hkv, d, rows, window):
    """Few enough splits to be joined inside one launch; sequences that need fewer of them, or none."""
    for lens in ([1300], [1290, 3, 700], [0, 1100]):
        _attend(paged, lens, [rows] * len(lens), hq, hkv, d, 32, window=window, one=rows == 1)


def test_peaked_and_flat_scores(paged):
    _attend(paged, [700, 1500], [1, 1], 4, 1, 64, 64, scale=6.0, one=True)
    _attend(paged, [700, 1500], [1, 1], 4, 1, 64, 64, scale=1e-4, one=True)
    _attend(paged, [200, 90], [70, 20], 4, 1, 64, 64, scale=4.0)


def test_pages_outside_the_cache_are_masked(paged):
    lens, page = [200, 90], 32
    pages, table = _filled(paged, lens, 2, 64, page)
    table[0][1], table[0][4], table[1][0] = -1, 1 << 20, pages.shape[0]
    q = _randn(4, 2, 8, 64).bfloat16().cuda()
    got = paged.kv4_attention(q, pages, torch.tensor(table, dtype=torch.int32).cuda(),
                              torch.tensor(lens, dtype=torch.int32).cuda())
    k, v = held(pages, 64)
    assert_attention(got, *plain_attention(q, k, v, table, lens, [0, 1, 2], 0.125, 0))


def test_lengths_and_rows_outside_the_tensors(paged):
    """Lengths past the table end there; offsets past q claim no rows: nothing is read or written outside."""
    pages, table = _filled(paged, [64, 64], 1, 64, 32)
    t = torch.tensor(table, dtype=torch.int32).cuda()
    q = _randn(4, 3, 4, 64).bfloat16().cuda()
    full = paged.kv4_attention(q[:2], pages, t, torch.tensor([64, 64], dtype=torch.int32).cuda())
    got = paged.kv4_attention(q[:2], pages, t, torch.tensor([64, 1 << 30], dtype=torch.int32).cuda())
    assert torch.equal(full, got)
    got = paged.kv4_attention(q[:2], pages, t, torch.tensor([64, -5], dtype=torch.int32).cuda())
    assert torch.equal(full[0], got[0]) and (got[1] == 0).all()
    out = torch.full_like(q, 7.0)
    cu = torch.tensor([0, 1, 1 << 30], dtype=torch.int32).cuda()
    paged.kv4_attention(q, pages, t, torch.tensor([64, 64], dtype=torch.int32).cuda(), cu, max_q=1, out=out)
    assert torch.equal(out[0], full[0]) and (out[2] == 7.0).all()
    cu = torch.tensor([-9, -3, 1], dtype=torch.int32).cuda()
    out.fill_(7.0)
    paged.kv4_attention(q, pages, t, torch.tensor([64, 64], dtype=torch.int32).cuda(), cu, max_q=4, out=out)
    assert (out[1:] == 7.0).all()


def test_nan_stays_where_it_is_seen(paged):
    """A stored NaN reaches the rows that see its key and no others, in the same call and sequence."""
    lens, page = [40], 16
    pages, table = _filled(paged, lens, 1, 64, page)
    bad = torch.full((1, 1, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    paged.kv4_append(None, bad, bad, pages, torch.tensor([table[0][2] * page + 5]).cuda())   # key 37
    q = _randn(4, 6, 4, 64).bfloat16().cuda()
    t, n = torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    cu = torch.tensor([0, 6], dtype=torch.int32).cuda()
    got = paged.kv4_attention(q, pages, t, n, cu, max_q=6)      # rows at positions 34 .. 39
    assert torch.isfinite(got[:3].float()).all() and torch.isnan(got[3:].float()).all()
    got = paged.kv4_attention(q, pages, t, n, cu, max_q=6, window=2)
    assert torch.isnan(got[3:5].float()).all() and torch.isfinite(got[[0, 1, 2, 5]].float()).all()
    q = _randn(5, 20, 4, 64).bfloat16().cuda()                  # positions 20 .. 39
    cu = torch.tensor([0, 20], dtype=torch.int32).cuda()
    got = paged.kv4_attention(q, pages, t, n, cu, max_q=20)
    assert torch.isfinite(got[:17].float()).all() and torch.isnan(got[17:].float()).all()
    # a value that is none in 32 of its dims, its key sound: those dims only
    good, half = torch.ones_like(bad), torch.ones_like(bad)
    half[..., 40] = float("inf")
    paged.kv4_append(None, good, half, pages, torch.tensor([table[0][2] * page + 5]).cuda())
    for rows, window in ((6, 0), (20, 0), (20, 2)):
        got = paged.kv4_attention(q[:rows], pages, t, n, torch.tensor([0, rows], dtype=torch.int32).cuda(), max_q=rows,
                                  window=window).float()
        sees = torch.zeros(rows, dtype=torch.bool)
        sees[rows - 3:rows - 1 if window else rows] = True
        assert torch.isfinite(got[..., :32]).all() and torch.isfinite(got[~sees]).all()
        assert torch.isnan(got[sees][..., 32:]).all()


def test_strided_queries_streams_and_repeats(paged):
    """Queries inside a wider tensor, another stream, twice the same bits."""
    lens = [900, 333, 1200]
    pages, table = _filled(paged, lens, 2, 64, 64)
    t, n = torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    wide = _randn(2, 3, 8 + 4, 2 * 64).bfloat16().cuda()
    q = wide[:, 2:10, 64:]
    ref = paged.kv4_attention(q.contiguous(), pages, t, n)
    assert torch.equal(paged.kv4_attention(q, pages, t, n), ref)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fresh = _filled(paged, lens, 2, 64, 64)[0]     # written and read on the side stream alone
        got = paged.kv4_attention(q, fresh, t, n)
    side.synchronize()
    assert torch.equal(got, ref)


def test_large_cache_offsets(paged):
    """A cache past 2^32 bytes: its last pages are written, read and attended at their own place."""
    page, d, hkv = 128, 128, 4
    per = hkv * paged.kv4_page_bytes(d, page)
    num = (1 << 32) // per + 3
    pages = torch.empty(num, hkv, per // hkv, dtype=torch.uint8, device="cuda")
    pages[-3:].fill_(0xFF)
    k, v = (_randn(i, 200, hkv, d).bfloat16().cuda() for i in (1, 2))
    at = torch.arange(200)
    where = torch.tensor([num - 1, num - 3])
    paged.kv4_append(None, k, v, pages, (where[at // page] * page + at % page).cuda())
    small = torch.full((3, hkv, per // hkv), 0xFF, dtype=torch.uint8, device="cuda")
    paged.kv4_append(None, k, v, small, (torch.tensor([2, 0])[at // page] * page + at % page).cuda())
    assert torch.equal(pages[-3:], small)
    q = _randn(3, 1, 8, d).bfloat16().cuda()
    n = torch.tensor([200], dtype=torch.int32).cuda()
    big = paged.kv4_attention(q, pages, where.int()[None].cuda(), n)
    assert torch.equal(big, paged.kv4_attention(q, small, torch.tensor([[2, 0]], dtype=torch.int32).cuda(), n))


def test_graph_replays_follow_lengths_and_slots(paged):
    """A decode step captured once (append, attention in splits with their merge) serves later steps: slots,
    positions, lengths and inputs are read on the device."""
    B, hq, hkv, d, page, width = 24, 16, 4, 64, 64, 40
    pages = paged.kv4_pages(B * width, hkv, d, page)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(1)).int().view(B, width).cuda()
    start = torch.randint(1500, 2500, (B,), generator=torch.Generator().manual_seed(2)).cuda()
    old = torch.arange(2500, device="cuda").repeat(B, 1)
    slots = torch.where(old < start[:, None], table.long().gather(1, old // page) * page + old % page, -1).flatten()
    k, v = (_randn(i, B * 2500, hkv, d).cuda().bfloat16() for i in (3, 4))
    paged.kv4_append(None, k, v, pages, slots)
    cos, sin = paged.rope_tables(width * page)
    qkv = [_randn(10 + i, B, hq + 2 * hkv, d).cuda().bfloat16() for i in range(3)]
    x, lens, slot = qkv[0].clone(), start.int(), torch.empty(B, dtype=torch.int64, device="cuda")

    def step():
        torch.add(table.long().gather(1, (lens.long() // page)[:, None])[:, 0] * page, lens.long() % page, out=slot)
        q = paged.kv4_append(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], pages, slot, lens, cos, sin)
        lens.add_(1)
        return paged.kv4_attention(q, pages, table, lens)

    empty = pages.clone()
    want = []
    for i in range(3):
        x.copy_(qkv[i])
        want.append(step())
    pages.copy_(empty)
    lens.copy_(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    pages.copy_(empty)
    lens.copy_(start)
    for i in range(3):
        x.copy_(qkv[i])
        graph.replay()
        assert torch.equal(got, want[i])


# -------------------------------------------------------------------------------------- refusals
def test_refusals(paged):
    pages = paged.kv4_pages(4, 2, 64, 16)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3, device="cuda")
    cos, sin = paged.rope_tables(8)
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")

    def refuse(match, f, *a, **k):
        with pytest.raises(RuntimeError, match=match):
            f(*a, **k)

    refuse("bfloat16", paged.kv4_append, x.float(), x, x, pages, slots)
    refuse("cache", paged.kv4_append, x, x[:, :1], x[:, :1], pages, slots)
    refuse("slots", paged.kv4_append, x, x, x, pages, slots.int())
    refuse("3 elements", paged.kv4_append, x, x, x, pages, slots[:2])
    refuse("positions", paged.kv4_append, x, x, x, pages, slots, None, cos, sin)
    refuse("multiple of 16", paged.kv4_append, x, x, x, pages, slots, pos, cos[:, :4].contiguous(),
           sin[:, :4].contiguous())
    refuse("q_norm", paged.kv4_append, x, x, x, pages, slots, q_norm=torch.ones(3, 64, device="cuda"))
    refuse("stride", paged.kv4_append, x, x.transpose(0, 2).contiguous().transpose(0, 2), x, pages, slots)
    refuse("page", paged.kv4_append, x, x, x, pages[..., :1000].contiguous(), slots)
    refuse("uint8", paged.kv4_read, pages.int(), slots)
    refuse("head_dim", paged.kv4_read, pages, slots, 96)
    table = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    refuse("query heads", paged.kv4_attention, x[:, :1], pages, table, lens)
    refuse("int32", paged.kv4_attention, x, pages, table.long(), lens)
    refuse("kv_lens", paged.kv4_attention, x, pages, table, lens[:2])
    refuse("one row", paged.kv4_attention, x[:2], pages, table, lens)
    refuse("max_q", paged.kv4_attention, x, pages, table, lens, max_q=2)
    refuse("out", paged.kv4_attention, x, pages, table, lens, out=x.float())
    refuse("window", paged.kv4_attention, x, pages, table, lens, window=-1)


def test_scale_is_positive_and_finite(paged):
    pages = paged.kv4_pages(4, 2, 64, 16)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    table, lens = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="scale"):
            paged.kv4_attention(x, pages, table, lens, scale=scale)
