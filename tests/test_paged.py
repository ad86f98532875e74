"""The paged 4-bit cache's operators on the CPU: what their C entry points and Python wrappers refuse (no GPU needed),
and the plain statement of a step's block tables against a known answer."""

import ctypes

import pytest
import torch

from locals_b200 import _lib, paged, rotary
from tests import paged_reference as R

OK = ctypes.c_void_p(4096)  # never dereferenced: argument checks come first


def test_plan_known_answer():
    # request 0 holds 5 of page 7's 8 places and brings 4; request 1 starts; request 2 brings nothing
    table, lens, q_start, positions, slots, head = R.plan([5, 0, 9], [4, 2, 0], [[7, -1], [-1, -1], [3, 4]],
                                                          [20, 21, 22], 1, 8, 7)
    assert table == [[7, 21], [22, -1], [3, 4]] and lens == [9, 2, 9] and q_start == [0, 4, 6, 6]
    assert positions == [5, 6, 7, 8, 0, 1, 0] and slots == [61, 62, 63, 168, 176, 177, -1] and head == 3


def test_rotary_tables_and_sections():
    cos, sin = rotary.tables(3, 4, 100.0, "cpu")
    angle = torch.tensor([[0.0, 0.0], [1.0, 0.1], [2.0, 0.2]], dtype=torch.float64)
    assert torch.equal(cos, angle.cos().float()) and torch.equal(sin, angle.sin().float())
    assert rotary.sections((1, 0, 2), "cpu").tolist() == [0, 2, 2]


def test_plan_refusals():
    L = _lib.lib()

    def rc(cached=OK, head=OK, head_out=ctypes.c_void_p(8192), B=2, width=4, nfree=3, page=16, tokens=5, lens=OK):
        return L.lq_page_plan(cached, OK, B, OK, width, OK, nfree, head, page, tokens, lens, OK, OK, OK, head_out, None)

    assert rc(cached=None) == _lib.LQ_E_ARG
    assert rc(head_out=OK) == _lib.LQ_E_ARG  # the head may not be its own successor
    for bad in (dict(B=0), dict(B=8193), dict(width=0), dict(nfree=-1), dict(page=0), dict(page=12), dict(tokens=-1)):
        assert rc(**bad) == _lib.LQ_E_SHAPE, bad
    assert rc(lens=ctypes.c_void_p(4098)) == _lib.LQ_E_ALIGN


def test_rotary_refusals():
    L = _lib.lib()

    def rc(q=OK, H=4, k=OK, KVH=2, N=3, D=64, rot=64, q_row=None, cos=OK, far=9, naxes=1, dtype=_lib.BF16):
        return L.lq_rotary(q, H * D if q_row is None else q_row, OK, H, k, KVH * D, OK, KVH, N, D, rot, OK, cos, OK, far,
                           None, naxes, 0, dtype, None)

    assert rc(q=None) == _lib.LQ_E_ARG
    assert rc(k=None) == _lib.LQ_E_ARG
    assert rc(cos=None) == _lib.LQ_E_ARG
    assert rc(dtype=_lib.F32) == _lib.LQ_E_UNSUPPORTED
    for bad in (dict(N=-1), dict(H=0, KVH=0), dict(rot=0), dict(rot=63), dict(rot=66), dict(far=0), dict(naxes=0),
                dict(q_row=4 * 64 - 1)):
        assert rc(**bad) == _lib.LQ_E_SHAPE, bad
    assert rc(q=ctypes.c_void_p(4097)) == _lib.LQ_E_ALIGN


def test_append_refusals():
    L = _lib.lib()

    def rc(k=OK, H=4, KVH=2, N=3, D=128, rot=128, pos=OK, cos=OK, k_row=None, pages=4, page=16, dtype=_lib.F16, kq=OK,
           q=OK):
        return L.lq_kv4_append(q, H * D, OK, H, k, KVH * D if k_row is None else k_row, OK, KVH * D, KVH, N, D, rot, pos,
                               cos, OK, 9, None, 1, 0, OK, kq, OK, OK, OK, OK, OK, pages, page, dtype, None)

    assert rc(k=None) == _lib.LQ_E_ARG
    assert rc(q=None) == _lib.LQ_E_ARG
    assert rc(cos=None) == _lib.LQ_E_ARG
    assert rc(dtype=_lib.F32) == _lib.LQ_E_UNSUPPORTED
    for bad in (dict(D=96), dict(rot=24), dict(page=12), dict(page=0), dict(pages=0), dict(KVH=0), dict(N=-1),
                dict(k_row=128), dict(pages=1 << 20, page=4096), dict(pages=1 << 26, page=16, KVH=5)):
        assert rc(**bad) == _lib.LQ_E_SHAPE, bad
    assert rc(k_row=2 * 128 + 4) == _lib.LQ_E_ALIGN
    assert rc(kq=ctypes.c_void_p(4104)) == _lib.LQ_E_ALIGN


def test_attend_and_read_refusals():
    L = _lib.lib()

    def rc(q=OK, N=3, q_start=OK, max_q=2, B=2, H=8, KVH=2, D=128, page=16, pages=4, width=4, window=0, scale=0.1,
           dtype=_lib.BF16, out=OK):
        return L.lq_kv4_attend(q, N, q_start, max_q, OK, OK, OK, OK, OK, OK, pages, page, OK, width, OK, B, None,
                               ctypes.c_float(scale), window, H, KVH, D, dtype, None, 0, out, None)

    assert rc(q=None) == _lib.LQ_E_ARG
    assert rc(dtype=_lib.F32) == _lib.LQ_E_UNSUPPORTED
    for bad in (dict(N=-1), dict(max_q=0), dict(B=0), dict(H=9), dict(H=0), dict(D=80), dict(page=20), dict(width=0),
                dict(window=-1), dict(scale=float("nan")), dict(q_start=None)):
        assert rc(**bad) == _lib.LQ_E_SHAPE, bad
    assert rc(out=ctypes.c_void_p(4098)) == _lib.LQ_E_ALIGN
    assert L.lq_kv4_read(OK, OK, OK, OK, OK, OK, 4, 16, 2, 128, None, 3, OK, OK, _lib.BF16, None) == _lib.LQ_E_ARG
    assert L.lq_kv4_read(OK, OK, OK, OK, OK, OK, 4, 16, 2, 96, OK, 3, OK, OK, _lib.BF16, None) == _lib.LQ_E_SHAPE


def test_wrappers_refuse_tensors_that_are_not_on_the_gpu_or_do_not_fit():
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    cos, sin = rotary.tables(4, 64, device="cpu")
    with pytest.raises(ValueError):
        paged.plan(i, i, i.view(2, 1), i, i[:1], 16, 2)
    with pytest.raises(ValueError):
        rotary.rotate(x, None, i, cos, sin)
    with pytest.raises(ValueError):
        rotary.rotate(x[0], None, i, cos, sin)
    with pytest.raises(ValueError):
        paged.pool(4, 2, 12, 128, device="cpu")
    with pytest.raises(ValueError):
        paged.pool(4, 2, 16, 80, device="cpu")
    keys, values = paged.pool(4, 4, 16, 64, torch.bfloat16, "cpu")
    with pytest.raises(ValueError):
        paged.append(x, x, x, i, keys, values)
    with pytest.raises(ValueError):
        paged.attend(x, keys, values, i.view(2, 1), i, 0.1)
    with pytest.raises(ValueError):
        paged.read(keys, values, i)
