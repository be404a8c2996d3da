"""The paged 4-bit KV cache without a GPU: argument checks of the C entries and of the Python functions,
sizes, rotation tables."""

from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from pulsar_b200 import _lib, build, paged


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_page_bytes():
    assert paged.kv4_page_bytes(64, 64) == 5120 and paged.kv4_page_bytes(128, 16) == 2560
    for hd, page in ((96, 64), (64, 8), (64, 48), (64, 1 << 17)):
        with pytest.raises(RuntimeError):
            paged.kv4_page_bytes(hd, page)
    with pytest.raises(RuntimeError):
        paged.kv4_pages(0, 4, device="cpu")
    assert paged.kv4_pages(3, 2, 64, 32, device="cpu").shape == (3, 2, 2560)


def test_cpu_tensors_are_refused():
    pages, slots = paged.kv4_pages(2, 1, device="cpu"), torch.zeros(1, dtype=torch.int64)
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.kv4_append(x, x, x, pages, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.kv4_read(pages, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.kv4_attention(x, pages, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))


def test_rope_tables():
    cos, sin = paged.rope_tables(100, 32, 10000.0, device="cpu")
    assert cos.shape == sin.shape == (100, 16) and cos.dtype == torch.float32
    i, t = 5, 77
    angle = t * 10000.0 ** (-2 * i / 32)
    assert math.isclose(cos[t, i], math.cos(angle), abs_tol=1e-6) and math.isclose(sin[t, i], math.sin(angle), abs_tol=1e-6)
    lin = paged.rope_tables(100, 32, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(lin[0][80], cos[20]) and torch.equal(lin[1][80], sin[20])
    ntk = paged.rope_tables(100, 32, scaling="ntk", factor=4.0, device="cpu")
    assert torch.equal(ntk[0][:, 0], cos[:, 0])            # the fastest dims keep their frequency ...
    want = 10000.0 ** (-30 / 32) / 4                       # ... the slowest are stretched by the factor
    assert math.isclose(ntk[1][50, 15], math.sin(50 * want), rel_tol=1e-5)
    yarn = paged.rope_tables(100, 32, scaling="yarn", factor=4.0, base_len=1024, device="cpu")
    assert torch.equal(yarn[0][:, 0], cos[:, 0])           # 163 turns in 1024 positions: kept
    assert torch.allclose(yarn[1][:, 15], lin[1][:, 15], atol=1e-7)   # under one turn: stretched
    assert lin[1][50, 8] < yarn[1][50, 8] < sin[50, 8]     # in between: blended
    for bad in (dict(rot_dim=7), dict(scaling="other"), dict(factor=0.5), dict(max_pos=0)):
        with pytest.raises(RuntimeError):
            paged.rope_tables(**{"max_pos": 4, "rot_dim": 8, "device": "cpu", **bad})


def test_c_entries_check_their_arguments(lib):
    def bad(match, f, *a):
        assert f(*a) == -1 and match in _lib.last_error(), _lib.last_error()

    some = 1 << 20       # an aligned address that no call below gets as far as using
    ap, rd, at = lib.pulsar_op_kv4_append, lib.pulsar_op_kv4_read, lib.pulsar_op_kv4_attention
    strides = (C.c_int64 * 6)(1024, 64, 256, 64, 256, 64)

    def append(n=1, hd=64, rot=0, max_pos=0, inter=0, page=64, pages=some, st=strides, k=some, cos=None, pos=None,
               slots=some):
        return (some, k, some, st, n, 16, 4, hd, None, None, 1e-6, cos, cos, rot, max_pos, inter, None, pos, slots,
                pages, 8, page, some, None)

    bad("head_dim", ap, *append(hd=96))
    bad("page_size", ap, *append(page=24))
    bad("aligned", ap, *append(pages=some + 8))
    bad("multiple of 16", ap, *append(rot=24))
    bad("multiple of 2", ap, *append(rot=23, inter=1))
    bad("null pointer", ap, *append(k=None))
    bad("null rotation table", ap, *append(rot=64, max_pos=9, pos=some))
    bad("need positions", ap, *append(rot=64, max_pos=9, cos=some))
    bad("strides", ap, *append(st=(C.c_int64 * 6)(1024, 64, 256, 60, 256, 64)))
    bad("16-byte aligned", ap, *append(k=some + 2))
    bad("invalid shape", ap, *append(n=1 << 31))
    assert ap(*append(n=0)) == 0
    bad("null pointer", rd, some, 8, 64, 4, 64, None, 3, some, some, None)
    bad("invalid shape", rd, some, 8, 64, 4, 64, some, 1 << 31, some, some, None)
    assert rd(some, 8, 64, 4, 64, None, 0, None, None, None) == 0

    def attend(q=some, n=4, hq=16, hd=64, page=64, b=4, cu=None, max_q=1, max_kv=100, scale=0.125, window=0, ws=None,
               wsb=0, out=some, row=1024):
        return (q, row, 64, n, hq, hd, some, 8, page, 4, some, b, 2, some, cu, max_q, max_kv, scale, window, ws, wsb,
                out, None)

    bad("head_dim", at, *attend(hd=80))
    bad("query heads", at, *attend(hq=6))
    bad("page_size", at, *attend(page=17))
    bad("one row", at, *attend(n=5))
    bad("max_q", at, *attend(max_q=0))
    bad("window", at, *attend(window=-1))
    bad("scale", at, *attend(scale=0.0))
    bad("even strides", at, *attend(row=1023))
    bad("16-byte", at, *attend(out=some + 4))
    bad("null pointer", at, *attend(q=None))
    bad("workspace", at, *attend(max_kv=1 << 20))
    assert at(*attend(n=0, b=0)) == 0
    need = C.c_int64(-1)
    assert lib.pulsar_op_kv4_attention_workspace(4, 16, 4, 64, 4, 1, 100, 0, C.byref(need)) == 0 and need.value == 0
    assert lib.pulsar_op_kv4_attention_workspace(4, 16, 4, 64, 4, 1, 1 << 17, 0, C.byref(need)) == 0
    assert need.value > 0 and need.value % (4 * 16 * 66 * 4) == 0
