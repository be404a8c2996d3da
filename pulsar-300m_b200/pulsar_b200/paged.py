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
import math

import torch

from . import _lib

_BF16, _F32, _I32, _I64, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


def _vector(t, name, dtype, n, dev):
    _check(t.is_cuda and t.device == dev and t.dtype == dtype and t.dim() == 1 and t.is_contiguous(),
           f"{name} must be a contiguous 1-D {str(dtype)[6:]} tensor on {dev}")
    _check(n is None or t.shape[0] == n, f"{name} must have {n} elements, got {t.shape[0]}")


def kv4_page_bytes(head_dim: int = 64, page_size: int = 64) -> int:
    """Bytes of one kv head's part of a page: 20 * head_dim for every 16 tokens."""
    _check(head_dim in (64, 128), f"head_dim must be 64 or 128, got {head_dim}")
    _check(page_size >= 16 and page_size & (page_size - 1) == 0 and page_size <= 65536,
           f"page_size must be a power of two from 16 to 65536, got {page_size}")
    return 20 * head_dim * page_size // 16


def kv4_pages(num_pages: int, num_kv_heads: int, head_dim: int = 64, page_size: int = 64, device="cuda"):
    """An empty cache: uint8 [num_pages, num_kv_heads, kv4_page_bytes(head_dim, page_size)]."""
    _check(num_pages >= 1 and num_kv_heads >= 1, "a cache needs at least one page and one kv head")
    return torch.zeros(num_pages, num_kv_heads, kv4_page_bytes(head_dim, page_size), dtype=_U8, device=device)


def _cache(pages, head_dim):
    """(number of pages, kv heads, page size) of a cache tensor."""
    _check(pages.is_cuda and pages.dtype == _U8 and pages.dim() == 3 and pages.is_contiguous(),
           "pages must be a contiguous uint8 CUDA tensor [num_pages, kv heads, page bytes]")
    num, hkv, nbytes = pages.shape
    page_size = nbytes * 16 // (20 * head_dim) if head_dim else 0
    _check(head_dim in (64, 128), f"head_dim must be 64 or 128, got {head_dim}")
    _check(page_size >= 16 and page_size & (page_size - 1) == 0 and page_size * 20 * head_dim == nbytes * 16,
           f"a page of {nbytes} bytes is no power of two of tokens (at least 16) with head_dim {head_dim}")
    return num, hkv, page_size


def rope_tables(max_pos: int, rot_dim: int = 64, theta: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                base_len: int = 1024, beta_fast: float = 32.0, beta_slow: float = 1.0, device="cuda"):
    """(cos, sin), fp32 [max_pos, rot_dim / 2], angles computed in fp64.

    ``scaling`` stretches the rotation to contexts ``factor`` times ``base_len``: "linear" divides
    every frequency by ``factor``; "ntk" raises theta by factor ** (rot_dim / (rot_dim - 2)); "yarn"
    divides the frequencies that turn fewer than ``beta_slow`` times within ``base_len``, keeps those
    that turn more than ``beta_fast`` times, and blends in between.
    """
    _check(rot_dim >= 2 and rot_dim % 2 == 0, f"rot_dim must be even, got {rot_dim}")
    _check(scaling in ("none", "linear", "ntk", "yarn"), f"unknown scaling {scaling!r}")
    _check(factor >= 1.0 and max_pos >= 1, "factor and max_pos must be at least 1")
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
    _check(x.is_cuda and x.device == dev and x.dtype == _BF16 and x.dim() == 3,
           f"{name} must be a bfloat16 tensor [tokens, heads, head_dim] on {dev}")
    _check(x.shape[0] == n and x.shape[2] == hd, f"{name} must be [{n}, heads, {hd}], got {list(x.shape)}")
    _check(x.numel() == 0 or (x.stride(2) == 1 and x.stride(0) % 8 == 0 and x.stride(1) % 8 == 0
                              and x.data_ptr() % 16 == 0),
           f"{name} needs stride(-1) == 1, other strides a multiple of 8 and 16-byte alignment")


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
    _check(k.dim() == 3, "k must be [tokens, heads, head_dim]")
    n, hkv, hd = k.shape
    dev = pages.device
    num, cache_heads, page_size = _cache(pages, hd)
    _check(hkv == cache_heads, f"k has {hkv} heads, the cache {cache_heads}")
    _heads(k, "k", n, hd, dev)
    _heads(v, "v", n, hd, dev)
    _check(v.shape[1] == hkv, f"v has {v.shape[1]} heads, k {hkv}")
    hq = 0
    if q is not None:
        _heads(q, "q", n, hd, dev)
        hq = q.shape[1]
    _vector(slots, "slots", _I64, n, dev)
    rot = max_pos = 0
    if cos is not None:
        _check(sin is not None and cos.shape == sin.shape and cos.dim() == 2, "cos and sin must be [max_pos, rot / 2]")
        for x in (cos, sin):
            _check(x.is_cuda and x.device == dev and x.dtype == _F32 and x.is_contiguous(),
                   "cos and sin must be contiguous float32 tensors on the cache's device")
        max_pos, rot = cos.shape[0], 2 * cos.shape[1]
        _check(0 < rot <= hd and rot % (2 if interleaved else 16) == 0,
               f"rotated dims must be a multiple of {2 if interleaved else 16} up to {hd}, got {rot}")
    if q_gain is not None:
        _vector(q_gain, "q_gain", _F32, None, dev)
        _check(cos is None or q_gain.shape[0] == max_pos, "q_gain must have a factor for each row of cos")
        max_pos = q_gain.shape[0]
    if rot or q_gain is not None:
        _check(positions is not None and max_pos > 0, "rotation and q_gain need positions and non-empty tables")
        _vector(positions, "positions", _I32, n, dev)
    for w, name, heads in ((q_norm, "q_norm", hq), (k_norm, "k_norm", hkv)):
        _check(w is None or (w.is_cuda and w.device == dev and w.dtype == _F32 and w.is_contiguous()
                             and w.shape == (heads, hd)),
               f"{name} must be a contiguous float32 tensor [{heads}, {hd}] on the cache's device")
    out = torch.empty(n, hq, hd, dtype=_BF16, device=dev) if q is not None else None
    if n:
        st = (C.c_int64 * 6)(*((q.stride(0), q.stride(1)) if hq else (0, 0)), k.stride(0), k.stride(1), v.stride(0),
                             v.stride(1))
        with torch.cuda.device(dev):
            _lib.call("pulsar_op_kv4_append", _p(q), _p(k), _p(v), st, n, hq, hkv, hd, _p(q_norm), _p(k_norm), eps,
                      _p(cos), _p(sin), rot, max_pos, int(interleaved), _p(q_gain), _p(positions), _p(slots),
                      _p(pages), num, page_size, _p(out), _stream(pages))
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
        with torch.cuda.device(dev):
            _lib.call("pulsar_op_kv4_read", _p(pages), num, page_size, hkv, head_dim, _p(slots), n, _p(k), _p(v),
                      _stream(pages))
    return k, v


def kv4_attention(q, pages, block_table, kv_lens, cu_q=None, *, max_q: int = 1, max_kv: int | None = None,
                  scale: float | None = None, window: int = 0, out=None):
    """softmax(scale q k^T) v of each query row over its sequence's cached keys, bf16 [N, Hq, D].

    q: bf16 [N, Hq, D], last stride 1, other strides even. block_table: int32 [B, width] page numbers,
    kv_lens: int32 [B] keys of each sequence, the rows' own included. Rows cu_q[b] .. cu_q[b + 1] - 1
    (int32 [B + 1], at most ``max_q`` each) are the last ones of sequence b: row j of n sees the keys
    up to position kv_lens[b] - n + j, with ``window`` > 0 the last ``window`` of these. Without cu_q
    there is one row for each sequence. ``max_kv`` bounds kv_lens (default: the table's width); it only
    decides how the work is split. ``scale`` defaults to D ** -0.5.

    A row that sees no key is zero. Lengths past the table end there; pages numbered outside the cache
    are left out as if masked; rows that no sequence claims are not written.
    """
    _check(q.is_cuda and q.dtype == _BF16 and q.dim() == 3, "q must be a bfloat16 CUDA tensor [rows, heads, head_dim]")
    n, hq, hd = q.shape
    num, hkv, page_size = _cache(pages, hd)
    dev = pages.device
    _check(q.device == dev, f"q is on {q.device}, the cache on {dev}")
    _check(q.numel() == 0 or (q.stride(2) == 1 and q.stride(0) % 2 == 0 and q.stride(1) % 2 == 0
                              and q.data_ptr() % 4 == 0),
           "q needs stride(-1) == 1, even strides and 4-byte alignment")
    _check(hq >= hkv and hq % hkv == 0, f"{hq} query heads over {hkv} kv heads")
    _check(block_table.is_cuda and block_table.device == dev and block_table.dtype == _I32 and block_table.dim() == 2
           and block_table.is_contiguous(), "block_table must be a contiguous int32 tensor [sequences, width]")
    b, width = block_table.shape
    _vector(kv_lens, "kv_lens", _I32, b, dev)
    if cu_q is None:
        _check(n == b and max_q == 1, f"without cu_q every sequence has one row (max_q 1): {n} rows of {b} sequences")
    else:
        _vector(cu_q, "cu_q", _I32, b + 1, dev)
    _check(max_q >= 1 and window >= 0, "max_q must be at least 1, window at least 0")
    if max_kv is None:
        max_kv = max(1, width * page_size)
    _check(max_kv >= 1, "max_kv must be at least 1")
    if out is None:
        out = torch.empty(n, hq, hd, dtype=_BF16, device=dev)
    else:
        _check(out.is_cuda and out.device == dev and out.dtype == _BF16 and out.shape == q.shape
               and out.is_contiguous(), "out must be a contiguous bfloat16 tensor of q's shape")
    if n and b:
        need = C.c_int64()
        _lib.call("pulsar_op_kv4_attention_workspace", n, hq, hkv, hd, b, max_q, max_kv, window, C.byref(need))
        ws = torch.empty(need.value, dtype=_U8, device=dev) if need.value else None
        with torch.cuda.device(dev):
            _lib.call("pulsar_op_kv4_attention", _p(q), q.stride(0), q.stride(1), n, hq, hd, _p(pages), num, page_size,
                      hkv, _p(block_table), b, width, _p(kv_lens), _p(cu_q), max_q, max_kv,
                      hd ** -0.5 if scale is None else scale, window, _p(ws), need.value, _p(out), _stream(pages))
    return out
