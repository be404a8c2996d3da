"""Paged KV cache held in 4 bits: append (with the norm of each query and key head and the position
rotation), read, and attention over it, as functions on torch tensors.

The cache is one uint8 tensor ``pages`` of shape [num_pages, kv heads, page bytes] from
``kv4_pages``; a page holds ``page_size`` tokens of every kv head at 5 bits a dim (4-bit codes, and a
bf16 scale and minimum for each 32 dims), 3.2 times less than bf16. A token is addressed by its slot,
``page * page_size + place in the page``; a sequence by a row of a block table of page numbers. Which
page belongs to which sequence is the caller's to decide, so sequences grow a page at a time, share
pages of a common prefix and roll back by a shorter length.

Kernels run on torch's current stream; results are new tensors on the inputs' device; argument errors
raise ``RuntimeError``. Values on the device (slots, lengths, page numbers, row offsets) are not
checked on the host: the kernels hold every access inside the tensors (each function says how).
"""

from __future__ import annotations

import ctypes as C
import functools
import math

import torch

from . import _lib

_BF16, _F32, _I32, _I64, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8


def _refuse(msg: str):
    raise RuntimeError(msg)


def _p(t):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=64)
def _strides(*of):
    return (C.c_int64 * len(of))(*of)


# The current stream's handle; torch's own function for it, where it has one, costs 2 us less than
# building a Stream object, as much as a small kernel takes. A CUDA tensor is there when they are
# asked, so torch's state is set up.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_entries: dict = {}


def _call(name, dev, *args):
    """The library's entry point on dev's current stream, with dev current."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    index = dev.index
    stream = _raw_stream(index) if _raw_stream else torch.cuda.current_stream(dev).cuda_stream
    if _current_device() == index:
        status = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            status = fn(*args, stream)
    if status:
        _lib.check(status, name)


# The checks below run before every launch of a few microseconds: conditions first, texts only when
# they fail.
def _vector(t, name, dtype, n, dev):
    if t.dtype != dtype or t.dim() != 1 or t.device != dev or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous 1-D {str(dtype)[6:]} tensor on {dev}")
    if n is not None and t.shape[0] != n:
        _refuse(f"{name} must have {n} elements, got {t.shape[0]}")


def _check_page(head_dim, page_size):
    if head_dim not in (64, 128):
        _refuse(f"head_dim must be 64 or 128, got {head_dim}")
    if page_size < 16 or page_size & (page_size - 1) or page_size > 65536:
        _refuse(f"page_size must be a power of two from 16 to 65536, got {page_size}")


def kv4_page_bytes(head_dim: int = 64, page_size: int = 64) -> int:
    """Bytes of one kv head's part of a page: 20 * head_dim for every 16 tokens."""
    _check_page(head_dim, page_size)
    return 20 * head_dim * page_size // 16


def kv4_pages(num_pages: int, num_kv_heads: int, head_dim: int = 64, page_size: int = 64, device="cuda"):
    """An empty cache: uint8 [num_pages, num_kv_heads, kv4_page_bytes(head_dim, page_size)]."""
    if num_pages < 1 or num_kv_heads < 1:
        _refuse("a cache needs at least one page and one kv head")
    return torch.zeros(num_pages, num_kv_heads, kv4_page_bytes(head_dim, page_size), dtype=_U8, device=device)


def _cache(pages, head_dim):
    """(number of pages, kv heads, page size) of a cache tensor."""
    if pages.dtype != _U8 or pages.dim() != 3 or not pages.is_cuda or not pages.is_contiguous():
        _refuse("pages must be a contiguous uint8 CUDA tensor [num_pages, kv heads, page bytes]")
    num, hkv, nbytes = pages.shape
    page_size = nbytes * 4 // (5 * head_dim) if head_dim > 0 else 0
    if head_dim not in (64, 128) or page_size < 16 or page_size & (page_size - 1) or page_size * 5 * head_dim != nbytes * 4:
        _refuse(f"pages of {nbytes} bytes a kv head: no cache of head_dim {head_dim} (64 or 128) with a power of two "
                "of tokens, at least 16, in a page")
    return num, hkv, page_size


def rope_tables(max_pos: int, rot_dim: int = 64, theta: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                base_len: int = 1024, beta_fast: float = 32.0, beta_slow: float = 1.0, device="cuda"):
    """(cos, sin), fp32 [max_pos, rot_dim / 2], angles computed in fp64.

    ``scaling`` stretches the rotation to contexts ``factor`` times ``base_len``: "linear" divides
    every frequency by ``factor``; "ntk" raises theta by factor ** (rot_dim / (rot_dim - 2)); "yarn"
    divides the frequencies that turn fewer than ``beta_slow`` times within ``base_len``, keeps those
    that turn more than ``beta_fast`` times, and blends in between.
    """
    if rot_dim < 2 or rot_dim % 2:
        _refuse(f"rot_dim must be even, got {rot_dim}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        _refuse(f"unknown scaling {scaling!r}")
    if factor < 1.0 or max_pos < 1:
        _refuse("factor and max_pos must be at least 1")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    if scaling == "ntk" and rot_dim > 2:
        theta = theta * factor ** (rot_dim / (rot_dim - 2))
    freq = theta ** (-i / rot_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        turns = base_len * freq / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    angle = torch.outer(torch.arange(max_pos, dtype=torch.float64), freq)
    return angle.cos().float().to(device), angle.sin().float().to(device)


def _heads(x, name, n, hd, dev):
    """Checks x [tokens, heads, head_dim] and gives (heads, token stride, head stride)."""
    if x.dtype != _BF16 or x.dim() != 3 or x.device != dev:
        _refuse(f"{name} must be a bfloat16 tensor [tokens, heads, head_dim] on {dev}")
    rows, heads, dims = x.shape
    if rows != n or dims != hd:
        _refuse(f"{name} must be [{n}, heads, {hd}], got {list(x.shape)}")
    st, sh, sd = x.stride()
    if n and heads and (sd != 1 or st % 8 or sh % 8 or x.data_ptr() % 16):
        _refuse(f"{name} needs stride(-1) == 1, other strides a multiple of 8 and 16-byte alignment")
    return heads, st, sh


def kv4_append(q, k, v, pages, slots, positions=None, cos=None, sin=None, *, q_norm=None, k_norm=None,
               eps: float = 1e-6, interleaved: bool = False, q_gain=None):
    """Stores the tokens' keys and values in the cache and returns their queries, ready to attend:
    one launch for the per-head RMS norm, the position rotation, the quantisation and the writes.

    q [N, Hq, D] (or None: nothing is returned), k and v [N, Hkv, D]: bf16, views of a fused
    projection included (last stride 1, the others multiples of 8). slots: int64 [N]; a token whose
    slot lies outside the cache (-1, say) is not stored. Two tokens of a call must not share a slot.
    positions: int32 [N], rows of cos and sin (fp32 [max_pos, rot / 2], ``rope_tables``), which rotate
    the first ``rot`` dims of queries and keys: pairs (i, i + rot / 2), rot a multiple of 16, or
    neighbours (2i, 2i + 1) when ``interleaved``; without tables nothing turns. A token whose position
    is outside the tables is not stored and its query is zero. q_norm [Hq, D], k_norm [Hkv, D]: fp32
    weights of the norm w x / sqrt(mean(x^2) + eps), before the rotation; None: no norm. q_gain: fp32
    [max_pos], a factor of the query of each position (the long-context temperature of YaRN layers).
    """
    if k.dim() != 3:
        _refuse("k must be [tokens, heads, head_dim]")
    n, _, hd = k.shape
    dev = pages.device
    num, cache_heads, page_size = _cache(pages, hd)
    hkv, kt, kh = _heads(k, "k", n, hd, dev)
    v_heads, vt, vh = _heads(v, "v", n, hd, dev)
    if hkv != cache_heads or v_heads != hkv:
        _refuse(f"k has {hkv} heads, v {v_heads}, the cache {cache_heads}")
    hq = qt = qh = 0
    out = None
    if q is not None:
        hq, qt, qh = _heads(q, "q", n, hd, dev)
        out = torch.empty(n, hq, hd, dtype=_BF16, device=dev)
    _vector(slots, "slots", _I64, n, dev)
    rot = max_pos = 0
    if cos is not None or sin is not None:
        if cos is None or sin is None or cos.dim() != 2 or cos.shape != sin.shape:
            _refuse("cos and sin must both be given, as [max_pos, rot / 2]")
        if cos.dtype != _F32 or sin.dtype != _F32 or cos.device != dev or sin.device != dev or not (
                cos.is_contiguous() and sin.is_contiguous()):
            _refuse(f"cos and sin must be contiguous float32 tensors on {dev}")
        max_pos, rot = cos.shape
        rot *= 2
        if not 0 < rot <= hd or rot % (2 if interleaved else 16):
            _refuse(f"rotated dims must be a multiple of {2 if interleaved else 16} up to {hd}, got {rot}")
    if q_gain is not None:
        _vector(q_gain, "q_gain", _F32, None if cos is None else max_pos, dev)
        max_pos = q_gain.shape[0]
    if rot or q_gain is not None:
        if positions is None or max_pos < 1:
            _refuse("rotation and q_gain need positions and tables that are not empty")
        _vector(positions, "positions", _I32, n, dev)
    for w, name, heads in ((q_norm, "q_norm", hq), (k_norm, "k_norm", hkv)):
        if w is not None and (w.dtype != _F32 or w.shape != (heads, hd) or w.device != dev or not w.is_contiguous()):
            _refuse(f"{name} must be a contiguous float32 tensor [{heads}, {hd}] on {dev}")
    if n:
        _call("pulsar_op_kv4_append", dev, _p(q), k.data_ptr(), v.data_ptr(), _strides(qt, qh, kt, kh, vt, vh), n, hq,
              hkv, hd, _p(q_norm), _p(k_norm), eps, _p(cos), _p(sin), rot, max_pos, int(interleaved), _p(q_gain),
              _p(positions), slots.data_ptr(), pages.data_ptr(), num, page_size, _p(out))
    return out


def kv4_read(pages, slots, head_dim: int = 64):
    """(k, v), bf16 [N, Hkv, head_dim]: what the cache holds for the given slots (int64 [N]); zeros for
    a slot outside it."""
    num, hkv, page_size = _cache(pages, head_dim)
    dev = pages.device
    _vector(slots, "slots", _I64, None, dev)
    n = slots.shape[0]
    k = torch.empty(n, hkv, head_dim, dtype=_BF16, device=dev)
    v = torch.empty_like(k)
    if n:
        _call("pulsar_op_kv4_read", dev, pages.data_ptr(), num, page_size, hkv, head_dim, slots.data_ptr(), n,
              k.data_ptr(), v.data_ptr())
    return k, v


@functools.lru_cache(maxsize=1024)
def _workspace(n, hq, hkv, hd, b, max_q, max_kv, window):
    need = C.c_int64()
    _lib.call("pulsar_op_kv4_attention_workspace", n, hq, hkv, hd, b, max_q, max_kv, window, C.byref(need))
    return need.value


def kv4_attention(q, pages, block_table, kv_lens, cu_q=None, *, max_q: int = 1, max_kv: int | None = None,
                  scale: float | None = None, window: int = 0, out=None):
    """softmax(scale q k^T) v of each query row over its sequence's cached keys, bf16 [N, Hq, D].

    q: bf16 [N, Hq, D], last stride 1, other strides even. block_table: int32 [B, width] page numbers,
    kv_lens: int32 [B] keys of each sequence, the rows' own included. Rows cu_q[b] .. cu_q[b + 1] - 1
    (int32 [B + 1], at most ``max_q`` each) are the last ones of sequence b: row j of n sees the keys
    up to position kv_lens[b] - n + j, with ``window`` > 0 the last ``window`` of these. Without cu_q
    there is one row for each sequence. ``max_kv`` bounds kv_lens (default: the table's width); it only
    decides how the work is split. ``scale`` defaults to D ** -0.5.

    Sums are in 32 bits. Up to 8 units (max_q times the heads of a group) operands are good to 2^-16, for
    values between 2^-50 and 2^37, queries below 2^67, products of a query and a key from 2^-50 up and a
    scale of at most 2^50 (checked). Above, queries, keys, values and weights are fp16
    numbers with powers of two taken out of a row's query, and of the keys and of the values of each step
    of 32 or 128 positions. They are good to 2^-12 of themselves or to 2^-34 of the largest of the step
    (queries of a row: 2^-28, weights: 2^-32), whichever is more, from 2^-100 up; the step's largest may be
    one that only later rows of the call see. Steps of values 2^80 below an earlier one lose more.

    A row that sees no key is zero. Lengths past the table end there; pages numbered outside the cache
    are left out as if masked; rows that no sequence claims are not written.
    """
    dev = pages.device
    if q.dtype != _BF16 or q.dim() != 3 or q.device != dev:
        _refuse(f"q must be a bfloat16 tensor [rows, heads, head_dim] on {dev}")
    n, hq, hd = q.shape
    num, hkv, page_size = _cache(pages, hd)
    qt, qh, qd = q.stride()
    if n and (qd != 1 or qt % 2 or qh % 2 or q.data_ptr() % 4):
        _refuse("q needs stride(-1) == 1, even strides and 4-byte alignment")
    if hq < hkv or hq % hkv:
        _refuse(f"{hq} query heads over {hkv} kv heads")
    if block_table.dtype != _I32 or block_table.dim() != 2 or block_table.device != dev or (
            not block_table.is_contiguous()):
        _refuse(f"block_table must be a contiguous int32 tensor [sequences, width] on {dev}")
    b, width = block_table.shape
    _vector(kv_lens, "kv_lens", _I32, b, dev)
    if cu_q is not None:
        _vector(cu_q, "cu_q", _I32, b + 1, dev)
    elif n != b or max_q != 1:
        _refuse(f"without cu_q every sequence has one row (max_q 1): {n} rows of {b} sequences")
    if max_kv is None:
        max_kv = max(1, width * page_size)
    if max_q < 1 or window < 0 or max_kv < 1:
        _refuse("max_q and max_kv must be at least 1, window at least 0")
    if scale is None:
        scale = hd ** -0.5
    elif not 0 < scale < math.inf:
        _refuse(f"scale must be positive and finite, got {scale}")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(n, hq, hd, dtype=_BF16, device=dev)
    elif out.dtype != _BF16 or out.shape != q.shape or out.device != dev or not out.is_contiguous():
        _refuse("out must be a contiguous bfloat16 tensor of q's shape")
    if n and b:
        need = _workspace(n, hq, hkv, hd, b, max_q, max_kv, window)
        ws = torch.empty(need, dtype=_U8, device=dev) if need else None
        _call("pulsar_op_kv4_attention", dev, q.data_ptr(), qt, qh, n, hq, hd, pages.data_ptr(), num, page_size, hkv,
              block_table.data_ptr(), b, width, kv_lens.data_ptr(), _p(cu_q), max_q, max_kv,
              scale, window, _p(ws), need, out.data_ptr())
    return out
