"""Attention over the paged 4-bit KV cache at its edges, against the definition in 64 bits.

Tolerance: a row's distance (2-norm over a head's dims) is at most 2^-8 of the row's own norm. Rounding
the result to bf16 moves it by 2^-9 at most. Above 8 units keys, values and weights are rounded at 2^-12:
with scale sum |q k| of a few units, random signs and Gaussian data that is some 2^-11.5 in the weights of a
row and 2^-12.5 each in values and weights, together 2^-11 of the row, a quarter of the other 2^-9. Up to 8 units
operands are good to 2^-16. A row that sees no key is exactly zero."""

from __future__ import annotations

import math

import pytest
import torch

from test_paged_kv4_gpu import held

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    from pulsar_b200 import paged
    return paged


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(paged, lens, k, v, page, seed=0):
    """The sequences' keys and values (bf16 [all keys, heads, D], one after the other) on shuffled pages;
    unused places hold NaN."""
    used = [-(-n // page) for n in lens]
    perm = torch.randperm(sum(used) + 1, generator=torch.Generator().manual_seed(seed)).tolist()
    width, table, slots = max(1, *used), [], []
    for n, u in zip(lens, used):
        mine = torch.tensor([perm.pop() for _ in range(u)] + [-1] * (width - u))
        at = torch.arange(n)
        table.append(mine.tolist())
        slots.append(mine[at // page] * page + at % page)
    pages = paged.kv4_pages(sum(used) + 1, k.shape[1], k.shape[2], page).fill_(0xFF)
    paged.kv4_append(None, k.bfloat16().cuda(), v.bfloat16().cuda(), pages, torch.cat(slots).cuda())
    return pages, table


def _exact(q, pages, table, lens, counts, scale, window):
    k, v = (x.cuda() for x in held(pages, q.shape[2]))
    page, out, row = k.shape[1], torch.zeros(q.shape, dtype=torch.double, device="cuda"), 0
    group = q.shape[1] // k.shape[2]
    for pages_b, n, c in zip(table, lens, counts):
        at = torch.arange(n, device="cuda")
        where = torch.tensor(pages_b, device="cuda")[at // page]
        at, where = (x[(where >= 0) & (where < len(k))] for x in (at, where))
        kk, vv = (x[where, at % page].repeat_interleave(group, 1) for x in (k, v))
        pos = n - c + torch.arange(c, device="cuda")[:, None]
        see = (at <= pos) & (at > pos - window if window else at >= 0)
        s = torch.einsum("qhd,khd->hqk", q[row:row + c].double(), kk) * scale
        s = s.masked_fill(~see, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300) if len(at) else s)
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        # a value that no row sees may be anything
        out[row:row + c] = torch.einsum("hqk,khd->qhd", p, torch.where(see.any(0)[:, None, None], vv, 0.0))
        row += c
    return out


def _attend(paged, q, pages, table, lens, counts, scale=None, window=0, **kw):
    """The kernel's answer, held against the definition."""
    cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    kw.setdefault("max_q", max(1, *counts))
    got = paged.kv4_attention(q, pages, _int(table), _int(lens), _int(cu), scale=scale, window=window, **kw)
    ref = _exact(q, pages, table, lens, counts, q.shape[2] ** -0.5 if scale is None else scale, window)
    assert torch.isfinite(got).all()
    err, size = (got.double() - ref).norm(dim=-1), ref.norm(dim=-1)
    assert (err[size == 0] == 0).all()
    worst = (err / size.clamp(min=1e-300)).max().item()
    assert worst <= 2.0 ** -8, f"a row is off by {worst:.3e} of its norm"
    return got


# Rows of a sequence, query heads, head dim, the bound of rows given: up to 8 units (query rows x heads of
# a group), above, and the kernel for many rows (chosen by a bound of rows that small calls do not fill).
KERNELS = [pytest.param(2, 4, 64, 2, id="few"), pytest.param(1, 7, 128, 1, id="few-128"),
           pytest.param(5, 4, 64, 5, id="wide"), pytest.param(3, 5, 128, 3, id="wide-128"),
           pytest.param(20, 4, 64, 8192, id="many"), pytest.param(20, 2, 128, 8192, id="many-128")]
ABOVE_8 = KERNELS[2:]


@pytest.mark.parametrize("rows,hq,d,max_q", KERNELS)
@pytest.mark.parametrize("qx,kx", [(0.0, 0.0), (0.0, 1.0), (2.0 ** -110, 2.0 ** -110)])
def test_queries_and_keys_of_zero(paged, rows, hq, d, max_q, qx, kx):
    """Scores of zero: the mean of the visible values, whatever is masked beside them. A query of zero is
    what an append gives for a position outside its tables, keys of zero what an empty cache holds."""
    lens, counts = [0, 1, 40, 300, 129], [rows, rows, rows, rows, 0]
    q = (_randn(1, sum(counts), hq, d) * qx).bfloat16().cuda()
    k, v = _randn(2, sum(lens), 1, d) * kx, _randn(3, sum(lens), 1, d)
    pages, table = _cache(paged, lens, k, v, 32)
    for window in (0, 3, 100):
        _attend(paged, q, pages, table, lens, counts, window=window, max_q=max_q)
    table[3][4:8] = [-1] * 4          # a whole step of 128 keys without a page
    table[2][0] = 1 << 20
    _attend(paged, q, pages, table, lens, counts, max_q=max_q)
    table[3] = [-1] * len(table[3])   # no page at all
    assert (_attend(paged, q, pages, table, lens, counts, max_q=max_q)[3 * rows:] == 0).all()


@pytest.mark.parametrize("rows,hq,d,max_q", KERNELS)
def test_queries_of_zero_on_an_empty_cache(paged, rows, hq, d, max_q):
    pages = paged.kv4_pages(8, 1, d, 32)
    q = torch.zeros(2 * rows, hq, d, dtype=torch.bfloat16, device="cuda")
    got = paged.kv4_attention(q, pages, _int([[0, 1, 2, 3], [4, 5, 6, 7]]), _int([100, 0]), _int([0, rows, 2 * rows]),
                              max_q=max_q)
    assert (got == 0).all()


@pytest.mark.parametrize("rows,hq,d,max_q", KERNELS)
@pytest.mark.parametrize("max_kv", [None, 64])
def test_one_key_above_a_flat_tail(paged, rows, hq, d, max_q, max_kv):
    """Every key of a long tail weighs half a millionth of the first one, whose value is zero: the tail's
    weights keep their precision (all of them are the same number, so roundings would not average out)."""
    n = 16384
    k, v = torch.zeros(n, 1, d), 1 + 0.5 * _randn(1, n, 1, d)
    k[0], v[0] = 1.0, 0.0
    pages, table = _cache(paged, [n], k, v, 64)
    q = torch.ones(rows, hq, d, dtype=torch.bfloat16, device="cuda")
    _attend(paged, q, pages, table, [n], [rows], scale=math.log(2.0 ** 24 / 8.45) / d, max_q=max_q, max_kv=max_kv)


@pytest.mark.parametrize("rows,hq,d,max_q", ABOVE_8)
@pytest.mark.parametrize("size,first", [(2.0 ** 20, 1), (2.0 ** 40, 128), (2.0 ** 70, 256)])
def test_large_values_of_no_weight(paged, rows, hq, d, max_q, size, first):
    """Values of a sequence's first keys, of hardly any weight, are many times larger than those that
    make the result: one key among others up to 2^20, whole steps of keys by any factor."""
    n = 1100
    base = _randn(1, 1, 1, d)
    q = (base + 0.1 * _randn(2, rows, hq, d)).bfloat16().cuda()
    k, v = _randn(3, n, 1, d), _randn(4, n, 1, d)
    k[:first] = -12 * base[0] - 0.1 * _randn(5, first, 1, d)
    v[:first] *= size
    pages, table = _cache(paged, [n], k, v, 64)
    for max_kv in (None, 64):
        _attend(paged, q, pages, table, [n], [rows], max_q=max_q, max_kv=max_kv)
    _attend(paged, q, pages, table, [n], [rows], max_q=max_q, window=900)


@pytest.mark.parametrize("rows,hq,d,max_q", ABOVE_8)
def test_values_that_grow_and_shrink(paged, rows, hq, d, max_q):
    """Steps of values of sizes between 2^-30 and 2^30, in turn: the largest ones make the result."""
    n = 1500
    k, v = _randn(3, n, 1, d), _randn(4, n, 1, d) * (2.0 ** (_randn(5, 12).clamp(-3, 3) * 10).round())[
        torch.arange(n) // 128][:, None, None]
    v[1200:1300] = 0.0
    pages, table = _cache(paged, [n], k, v, 16)
    q = _randn(1, rows, hq, d).bfloat16().cuda()
    for max_kv in (None, 64):
        _attend(paged, q, pages, table, [n], [rows], max_q=max_q, max_kv=max_kv)


@pytest.mark.parametrize("rows,hq,d,max_q", ABOVE_8)
@pytest.mark.parametrize("qx,kx,vx", [(1.0, 2.0 ** 120, 2.0 ** 120), (2.0 ** 115, 2.0 ** -90, 2.0 ** -90),
                                      (2.0 ** -90, 2.0 ** 100, 2.0 ** 118)])
def test_sizes_at_the_ends_of_the_type(paged, rows, hq, d, max_q, qx, kx, vx):
    lens, counts = [300, 40], [rows, rows]
    pages, table = _cache(paged, lens, _randn(1, 340, 1, d) * kx, _randn(2, 340, 1, d) * vx, 64)
    q = (_randn(3, 2 * rows, hq, d) * qx).bfloat16().cuda()
    _attend(paged, q, pages, table, lens, counts, scale=0.12 / qx / kx, max_q=max_q)


@pytest.mark.parametrize("rows,hq,d,max_q", ABOVE_8)
def test_a_large_value_that_only_the_last_row_sees(paged, rows, hq, d, max_q):
    """Above 8 units the values of a step of keys share a power of two, keys of later rows among them: values
    2^20 below the largest still have their precision."""
    n = 290
    v = _randn(2, n, 1, d)
    v[n - 1] *= 2.0 ** 20
    pages, table = _cache(paged, [n], _randn(1, n, 1, d), v, 64)
    _attend(paged, _randn(3, rows, hq, d).bfloat16().cuda(), pages, table, [n], [rows], max_q=max_q)


@pytest.mark.parametrize("rows,hq,d,max_q", KERNELS[:2])
@pytest.mark.parametrize("vx", [2.0 ** -47, 2.0 ** 34])
def test_sizes_up_to_8_units(paged, rows, hq, d, max_q, vx):
    """Up to 8 units values between 2^-50 and 2^37 keep their precision."""
    lens, counts = [300, 40], [rows, rows]
    pages, table = _cache(paged, lens, _randn(1, 340, 1, d), _randn(2, 340, 1, d) * vx, 64)
    _attend(paged, _randn(3, 2 * rows, hq, d).bfloat16().cuda(), pages, table, lens, counts, max_q=max_q)


def test_half_a_rotation_table_is_refused(paged):
    pages = paged.kv4_pages(4, 2, 64, 16)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    cos, sin = paged.rope_tables(8)
    for c, s in ((cos, None), (None, sin)):
        with pytest.raises(RuntimeError, match="cos and sin"):
            paged.kv4_append(x, x, x, pages, torch.arange(3, device="cuda"), _int([0, 1, 2]), c, s)


@pytest.mark.parametrize("hq,hkv,d,page,window", [(16, 4, 64, 64, 0), (28, 4, 64, 16, 50), (16, 4, 128, 32, 70),
                                                  (28, 4, 128, 64, 0), (4, 4, 64, 32, 1)])
def test_many_short_sequences(paged, hq, hkv, d, page, window):
    """More sequences and kv heads (640) than the GPU holds CTAs of four warps: blocks of two warps."""
    edges = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129]
    lens = (edges + torch.randint(301, (145,), generator=torch.Generator().manual_seed(1)).tolist())
    k, v = _randn(2, sum(lens), hkv, d), _randn(3, sum(lens), hkv, d)
    pages, table = _cache(paged, lens, k, v, page)
    for b in (40, 77, 120):
        table[b][0] = -1
    table[150] = [1 << 20] * len(table[150])
    q = (1.5 * _randn(4, 160, hq, d)).bfloat16().cuda()
    got = _attend(paged, q, pages, table, lens, [1] * 160, window=window, max_kv=300)
    one = paged.kv4_attention(q, pages, _int(table), _int(lens), window=window, max_kv=300)
    assert torch.equal(one, got)


@pytest.mark.parametrize("rows,hq,d,max_q", KERNELS)
@pytest.mark.parametrize("page,window", [(16, 0), (64, 0), (64, 4500)])
def test_long_walks(paged, rows, hq, d, max_q, page, window):
    """One CTA walks a whole sequence (max_kv far below the truth), so that pages are looked up again and
    again on the way; some are missing, late ones too."""
    lens, counts = [9000, 4200, 4097], [rows, rows, max(1, rows - 1)]
    pages, table = _cache(paged, lens, _randn(1, sum(lens), 1, d), _randn(2, sum(lens), 1, d), page)
    table[0][4500 // page], table[0][8500 // page], table[1][4150 // page], table[2][0] = -1, 1 << 20, -1, -1
    q = (1.2 * _randn(3, sum(counts), hq, d)).bfloat16().cuda()
    _attend(paged, q, pages, table, lens, counts, window=window, max_q=max_q, max_kv=64)


@pytest.mark.parametrize("rows,hq,hkv,d,page,window,max_q", [
    (65, 4, 1, 64, 64, 0, 65), (65, 4, 1, 64, 16, 70, 8192), (65, 8, 4, 128, 32, 0, 65), (65, 8, 4, 128, 32, 90, 8192),
    (8, 3, 3, 64, 128, 50, 8), (5, 7, 1, 128, 16, 33, 5), (6, 8, 2, 64, 32, 0, 6)])
def test_rows_by_their_norms(paged, rows, hq, hkv, d, page, window, max_q):
    """Prompts, chunks and verify blocks: a key too many or too few moves a row by more than the bound."""
    lens, counts = [150, 129, rows, 40, 0, 70], [rows, min(rows, 17), rows, 1, 2, 0]
    pages, table = _cache(paged, lens, 1.3 * _randn(1, sum(lens), hkv, d), _randn(2, sum(lens), hkv, d), page)
    q = (1.5 * _randn(3, sum(counts), hq, d)).bfloat16().cuda()
    _attend(paged, q, pages, table, lens, counts, window=window, max_q=max_q)


@pytest.mark.parametrize("rows,hq,d,max_q", KERNELS)
@pytest.mark.parametrize("window", [0, 5])
def test_large_scales(paged, rows, hq, d, max_q, window):
    """Keys of 2^-40 whose scale makes up for it; short sequences, rows that see no key."""
    lens, counts = [0, 1, 2, 40, 300], [rows] * 5
    k, v = _randn(1, sum(lens), 1, d) * 2.0 ** -40, _randn(2, sum(lens), 1, d)
    pages, table = _cache(paged, lens, k, v, 32)
    q = _randn(3, sum(counts), hq, d).bfloat16().cuda()
    _attend(paged, q, pages, table, lens, counts, scale=0.12 * 2.0 ** 40, window=window, max_q=max_q)


def test_scale_past_its_range_is_refused(paged):
    """Up to 8 units a scale past 2^50 would leave the range of the scores."""
    pages = paged.kv4_pages(4, 1, 64, 16)
    table, lens = _int([[0]] * 3), _int([1, 1, 1])
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    for scale in (2.0 ** 51, 1e30):
        with pytest.raises(RuntimeError, match="scale"):
            paged.kv4_attention(q, pages, table, lens, scale=scale)
    assert (paged.kv4_attention(q, pages, table, lens, scale=2.0 ** 50) == 0).all()
    assert (paged.kv4_attention(q, pages, table, lens, _int([0, 1, 2, 3]), max_q=3, scale=1e30) == 0).all()
