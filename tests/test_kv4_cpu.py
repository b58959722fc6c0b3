"""The 4-bit KV cache without a GPU: sizes, refusals of the entry points (made
before anything touches a device), and the tests' own reference."""
import ctypes as C

import numpy as np
import pytest

import kv4ref as R
import tinyminigo_amd as T
from tinyminigo_amd._lib import (
    TMG_E_CAPACITY, TMG_E_INVALID, TMG_OK, lib, tmg_kv4, tmg_kv4_attn_args,
)

A = 0x10000  # an address the refusals never follow


@pytest.mark.parametrize("cap,nkv,hd", [(1, 1, 16), (7, 2, 16), (5, 3, 32), (100, 2, 64), (512, 8, 128), (33, 4, 256)])
def test_slab_bytes(cap, nkv, hd):
    n = nkv * cap * (hd + 2 * R.groups(hd))
    assert T.kv4_bytes(cap, nkv, hd) == (n + 15) // 16 * 16


@pytest.mark.parametrize("cap,nkv,hd", [(0, 1, 64), (8, 0, 64), (8, 1, 0), (8, 1, 96), (8, 1, 512), (8, 40000, 64),
                                        (0x80000000, 1, 64)])
def test_slab_bytes_of_unsupported_shapes(cap, nkv, hd):
    assert T.kv4_bytes(cap, nkv, hd) == 0


def test_slab_bytes_past_32_bits():
    assert T.kv4_bytes(1 << 30, 8, 128) == (1 << 30) * 8 * 136


def kv(**over):
    d = dict(data=A, seq_stride=T.kv4_bytes(64, 2, 64), n_seq=3, cap=64, nkv=2, hd=64)
    d.update(over)
    return tmg_kv4(**d)


CACHES = [
    (dict(data=None), TMG_E_INVALID), (dict(data=A + 8), TMG_E_INVALID), (dict(hd=48), TMG_E_INVALID),
    (dict(nkv=0), TMG_E_INVALID), (dict(cap=0), TMG_E_INVALID), (dict(n_seq=65536), TMG_E_INVALID),
    (dict(seq_stride=T.kv4_bytes(64, 2, 64) - 16), TMG_E_INVALID),
    (dict(seq_stride=T.kv4_bytes(64, 2, 64) + 8), TMG_E_INVALID),
]
ROWS = [
    (dict(k=None), TMG_E_INVALID), (dict(k=A + 4), TMG_E_INVALID), (dict(v=A + 8), TMG_E_INVALID),
    (dict(stride=124), TMG_E_INVALID), (dict(stride=130), TMG_E_INVALID), (dict(pos=64), TMG_E_CAPACITY),
    (dict(pos=60, rows=5), TMG_E_CAPACITY), (dict(rows=65), TMG_E_CAPACITY), (dict(pos_dev=A + 2), TMG_E_INVALID),
    (dict(pos=0xFFFFFFFF, rows=2), TMG_E_CAPACITY), (dict(rows=65, pos_dev=A), TMG_E_CAPACITY),
]


def rows_call(fn, c, k=A, v=A, stride=0, rows=1, pos_dev=None, pos=0):
    return fn(C.byref(c) if c else None, k, v, stride, rows, pos_dev, pos, None)


@pytest.mark.parametrize("fn", ["tmg_kv4_write", "tmg_kv4_read"])
@pytest.mark.parametrize("over,code", CACHES)
def test_rows_refuse_caches(fn, over, code):
    assert rows_call(getattr(lib, fn), kv(**over)) == code
    assert lib.tmg_last_error()


@pytest.mark.parametrize("fn", ["tmg_kv4_write", "tmg_kv4_read"])
@pytest.mark.parametrize("over,code", ROWS)
def test_rows_refuse_rows(fn, over, code):
    if fn == "tmg_kv4_read" and over == dict(k=None):
        over = dict(k=None, v=None)  # one of the two may be left out
    assert rows_call(getattr(lib, fn), kv(), **over) == code


@pytest.mark.parametrize("fn", ["tmg_kv4_write", "tmg_kv4_read"])
def test_rows_nothing_to_do(fn):
    assert rows_call(getattr(lib, fn), kv(), rows=0) == TMG_OK
    assert rows_call(getattr(lib, fn), kv(n_seq=0)) == TMG_OK
    assert rows_call(getattr(lib, fn), None) == TMG_E_INVALID


def attn(c, **over):
    d = dict(q=A, out=A, k_new=None, v_new=None, q_stride=0, out_stride=0, new_stride=0, rows=1, nq=4, pos_dev=None,
             pos=3, scale=0.0, ws=A, ws_bytes=1 << 40)
    d.update(over)
    return lib.tmg_kv4_attn(C.byref(c) if c else None, C.byref(tmg_kv4_attn_args(**d)), None)


@pytest.mark.parametrize("over,code", CACHES)
def test_attn_refuses_caches(over, code):
    assert attn(kv(**over)) == code


@pytest.mark.parametrize("over,code", [
    (dict(q=None), TMG_E_INVALID), (dict(out=None), TMG_E_INVALID), (dict(q=A + 4), TMG_E_INVALID),
    (dict(out=A + 8), TMG_E_INVALID), (dict(nq=3), TMG_E_INVALID), (dict(nq=0), TMG_E_INVALID),
    (dict(nq=65538), TMG_E_INVALID), (dict(q_stride=252), TMG_E_INVALID), (dict(q_stride=257), TMG_E_INVALID),
    (dict(out_stride=252), TMG_E_INVALID), (dict(k_new=A), TMG_E_INVALID), (dict(v_new=A), TMG_E_INVALID),
    (dict(k_new=A, v_new=A + 4), TMG_E_INVALID), (dict(k_new=A, v_new=A, new_stride=64), TMG_E_INVALID),
    (dict(pos=64), TMG_E_CAPACITY), (dict(rows=65), TMG_E_CAPACITY), (dict(scale=float("nan")), TMG_E_INVALID),
    (dict(scale=float("inf")), TMG_E_INVALID), (dict(pos_dev=A + 1), TMG_E_INVALID),
])
def test_attn_refuses_arguments(over, code):
    assert attn(kv(), **over) == code


def test_attn_refuses_workspaces():
    c = kv(cap=4096, seq_stride=T.kv4_bytes(4096, 2, 64))
    n = C.c_size_t()
    assert lib.tmg_kv4_attn_workspace(C.byref(c), 1, 4, C.byref(n)) == TMG_OK
    assert n.value > 0
    for over in (dict(ws=None), dict(ws_bytes=n.value - 1), dict(ws=A + 4)):
        assert attn(c, **over) == TMG_E_INVALID
    assert lib.tmg_kv4_attn_workspace(C.byref(c), 1, 4, None) == TMG_E_INVALID
    assert lib.tmg_kv4_attn_workspace(C.byref(c), 1, 5, C.byref(n)) == TMG_E_INVALID
    assert lib.tmg_kv4_attn_workspace(C.byref(c), 4097, 4, C.byref(n)) == TMG_E_CAPACITY


def test_attn_nothing_to_do():
    assert attn(kv(), rows=0) == TMG_OK
    assert attn(kv(n_seq=0)) == TMG_OK
    assert attn(None) == TMG_E_INVALID
    assert lib.tmg_kv4_attn(C.byref(kv()), None, None) == TMG_E_INVALID


def test_too_many_rows_for_one_call():
    c = kv(cap=1 << 30, nkv=1, hd=256, n_seq=1)
    assert rows_call(lib.tmg_kv4_write, c, rows=(1 << 26) + 1) == TMG_E_INVALID
    assert attn(kv(cap=1 << 26, nkv=1, hd=16, n_seq=1), rows=1 << 26, nq=4, pos=0) == TMG_E_INVALID


def test_valid_calls_without_a_device():
    from tinyminigo_amd import hip as H
    from tinyminigo_amd._lib import TMG_E_DEVICE
    if H.device_count():
        pytest.skip("needs a machine without a GPU")
    assert rows_call(lib.tmg_kv4_write, kv()) == TMG_E_DEVICE
    assert rows_call(lib.tmg_kv4_read, kv()) == TMG_E_DEVICE
    assert attn(kv()) == TMG_E_DEVICE


def test_workspace_covers_every_position():
    # what a call at any position needs is within what the workspace query says
    for rows, nq, nkv, hd, cap, n_seq in [(1, 16, 8, 128, 131072, 1), (45, 16, 8, 128, 8192, 1), (1, 32, 8, 128, 4096, 48),
                                          (300, 4, 2, 16, 1000, 2), (1, 20, 1, 64, 500, 3)]:
        big = T.Kv4(A, cap=cap, nkv=nkv, hd=hd, n_seq=n_seq, seq_stride=T.kv4_bytes(cap, nkv, hd))
        most = T.kv4_attn_workspace(big, rows, nq)
        for c in (rows, rows + 1, (rows + cap) // 2):
            small = T.Kv4(A, cap=c, nkv=nkv, hd=hd, n_seq=n_seq, seq_stride=T.kv4_bytes(cap, nkv, hd))
            assert T.kv4_attn_workspace(small, rows, nq) <= most


def test_reference_rounds_to_nearest_even_code():
    x = np.zeros(32, np.float32)
    x[:14] = [7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 6.5, 0.2500001, 4.9999995, -7.0]
    code, byte = R.quantize(x)
    assert byte.tolist() == [127]
    assert R.values(code, byte)[:14].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -4, 6, 0.5, 4, -6]
    assert R.quantize(np.float32(7.0000005) * np.ones(32, np.float32))[1].tolist() == [128]
    assert R.quantize(np.zeros(32, np.float32))[1].tolist() == [27]
    y = np.ones(64, np.float32)
    y[40] = np.inf
    code, byte = R.quantize(y)
    assert byte[1] == 255 and np.isnan(R.values(code, byte)[32:]).all() and (R.values(code, byte)[:32] == 1).all()


def test_reference_error_is_half_a_spacing():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((200, 128)) * np.exp(rng.standard_normal((200, 1)))).astype(np.float32)
    code, byte = R.quantize(x)
    s = np.exp2(byte.astype(float) - 127).repeat(32, -1)
    a = np.abs(x) / s
    half = np.where(a <= 2, 0.25, np.where(a <= 4, 0.5, 1.0))
    assert (np.abs(x - R.values(code, byte)) <= half * s).all()
    assert (np.abs(x).reshape(200, 4, 32).max(-1) <= 7 * np.exp2(byte.astype(float) - 127)).all()
