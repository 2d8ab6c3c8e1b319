"""What the calls of the several-request step refuse, before anything is launched (no GPU needed)."""

import ctypes as C

import pytest

from drama_rs_b200 import ffi

A = 1 << 20  # an address that nothing reads: every call below is refused


def norms(o=A, o_type=0, post=A, gate=A, scale=A, x=A, x_out=A, pre=A, h=A, h_type=1, rows=1, d=2048):
    return ffi.lib().drb_block_norms(o, o_type, post, gate, scale, 1.0, x, x_out, pre, h, h_type, rows, d, 1e-6, None)


@pytest.mark.parametrize("kw", [dict(d=0), dict(d=8193), dict(rows=-1), dict(o_type=3), dict(o_type=-1), dict(h_type=3), dict(o=None), dict(x=None),
                                dict(x_out=None), dict(h=None)])
def test_norms_refuse_shapes_types_and_missing_buffers(kw):
    assert norms(**kw) == -1


@pytest.mark.parametrize("kw", [dict(o=A + 2), dict(o=A + 1, o_type=1), dict(x=A + 2), dict(x_out=A + 1), dict(h=A + 1), dict(h=A + 2, h_type=0), dict(gate=A + 2),
                                dict(post=A + 1), dict(scale=A + 3), dict(pre=A + 2)])
def test_norms_refuse_split_values(kw):
    assert norms(**kw) == -3


def few(w=None, x=A, y=A, live=None, n=4, e=64, topk=8, h=2048, i=512, ws=A):
    w = w or ffi.MoeLayerPtrs(*[A] * 10)
    return ffi.lib().drb_moe_few(C.byref(w), x, y, live, n, e, topk, h, i, 1e-6, ws, None)


@pytest.mark.parametrize("kw", [dict(n=17), dict(n=-1), dict(e=257), dict(e=7), dict(topk=0), dict(topk=9), dict(h=1024), dict(i=256), dict(x=None), dict(y=None),
                                dict(ws=None)])
def test_few_refuses_shapes_and_missing_buffers(kw):
    assert few(**kw) == -1


def test_few_refuses_missing_and_misaligned_weights():
    for j in range(10):
        for bad, code in ((None, -1), (A + 8, -3)):
            p = [A] * 10
            p[j] = bad
            assert few(w=ffi.MoeLayerPtrs(*p)) == code
    assert few(x=A + 4) == -3 and few(ws=A + 128) == -3 and few(y=A + 2) == -3
    assert ffi.lib().drb_moe_few(None, A, A, None, 4, 64, 8, 2048, 512, 1e-6, A, None) == -1


def test_few_workspace_sizes():
    ws = ffi.lib().drb_moe_few_workspace_bytes
    assert ws(0, 8) == -1 and ws(17, 8) == -1 and ws(1, 0) == -1 and ws(1, 9) == -1
    assert ws(16, 8) - ws(15, 8) >= 9 * (2048 + 512) * 4 and ws(1, 1) > 0


def lora(w=A, s=A, x=A, x_type=1, a=A, b=A, scale=A, who=A, adapters=2, rank=8, res=A, y=A, v=A, rows=4, n=64, k=512):
    return ffi.lib().drb_proj_q8_lora(w, s, x, x_type, a, b, scale, who, adapters, rank, res, y, v, rows, n, k, None)


@pytest.mark.parametrize("kw", [dict(x_type=0), dict(x_type=3), dict(rows=-1), dict(n=0), dict(k=0), dict(k=64), dict(k=200), dict(k=8320), dict(rank=72),
                                dict(rank=-8), dict(rank=12), dict(adapters=-1), dict(w=None), dict(s=None), dict(x=None), dict(y=None), dict(a=None),
                                dict(b=None), dict(scale=None), dict(who=None), dict(v=None)])
def test_lora_refuses_shapes_types_and_missing_buffers(kw):
    assert lora(**kw) == -1


@pytest.mark.parametrize("kw", [dict(w=A + 8), dict(s=A + 1), dict(x=A + 2), dict(a=A + 8), dict(b=A + 2), dict(v=A + 4), dict(y=A + 2), dict(res=A + 1),
                                dict(scale=A + 2), dict(who=A + 2)])
def test_lora_refuses_misaligned_buffers(kw):
    assert lora(**kw) == -3


def test_row_counts_have_a_limit():
    assert norms(rows=2**30 + 1) == -1 and norms(rows=2**31 - 1, d=1) == -1
    assert lora(rows=65535 * 64 + 1) == -1 and lora(rows=2**31 - 1) == -1
