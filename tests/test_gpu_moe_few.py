"""drb_moe_few (one MoE layer for 1 to 16 tokens) against the fp64 block.

Tolerance of a row, relative to its 2-norm, with u = 2^-24 and inputs of independent signs, whose roundings add up in quadrature: an input is
off by half a digit, at most u times the largest of 64 neighbours (3.5 times their rms at most here), and a sum over 2048 products meets three fp32 roundings
a group of 64, each of at most u times a partial sum: 3.5 u + sqrt(3 * 32) u < 13.4 u a projection. SwiGLU multiplies two of them (silu's slope
is below 1.1), down adds a third, the routing weights and the norm two of that size at most: 5 * 13.4 u = 4e-6.
"""

import ctypes as C

import numpy as np
import pytest

from drama_rs_b200 import ffi, synth
from drama_rs_b200.gpu import DevBuf, Graph, Stream, launched
from drama_rs_b200.model import MoeLayer
from oracle import moe_oracle as orc
from tests.helpers import device_error_word

pytestmark = pytest.mark.gpu
H, I, EPS = 2048, 512, 1e-6
REL = 4e-6


class Few:
    def __init__(self, host, n, topk, st):
        self.l, self.st, self.n, self.topk = ffi.lib(), st, n, topk
        self.dev = MoeLayer.upload(host, st)
        d = self.dev
        self.w = ffi.MoeLayerPtrs(*[t.ptr for t in (d.router, d.post_norm, d.gate_up.q, d.gate_up.sm, d.down.q, d.down.sm, d.shared_gate_up.q,
                                                    d.shared_gate_up.s, d.shared_down.q, d.shared_down.s)])
        self.ws = DevBuf.zeros(self.l.drb_moe_few_workspace_bytes(n, topk), st)

    def call(self, x, y, live=None, n=None, topk=None):
        return self.l.drb_moe_few(C.byref(self.w), x.at(0), y.at(0), live.at(0) if live is not None else None, self.n if n is None else n,
                                  self.dev.experts, self.topk if topk is None else topk, H, I, EPS, self.ws.at(0), self.st.raw)

    def run(self, x, live=None, in_place=False, topk=None):
        n = x.shape[0]
        dx = DevBuf.from_array(x.astype(np.float32), self.st)
        dy = dx if in_place else DevBuf.from_array(np.full((n, H), 7.0, np.float32), self.st)
        dl = DevBuf.from_array(np.asarray(live, np.uint8), self.st) if live is not None else None
        launched(self.call(dx, dy, dl, n, topk), "moe_few")
        return dy.download(np.float32, n * H, self.st).reshape(n, H)


def reference(host, x, topk):
    return orc.moe_layer(host, x, topk, EPS, np.float64)[0]


def assert_rows(y, ref, rows):
    for r in rows:
        rel = np.linalg.norm(y[r] - ref[r]) / np.linalg.norm(ref[r])
        assert rel <= REL, (r, rel)


_LAYERS = {}


def layer(e):
    if e not in _LAYERS:
        _LAYERS[e] = synth.make_layer(11 + e, synth.MoeShape(experts=e))
    return _LAYERS[e]


@pytest.mark.parametrize("e,n,topk", [(16, 1, 8), (16, 2, 8), (16, 3, 1), (16, 16, 8), (33, 5, 3), (8, 9, 8), (1, 4, 1), (1, 16, 1), (64, 8, 6),
                                      (64, 12, 2), (64, 7, 8), (64, 4, 8), (64, 13, 8), (8, 16, 8), (256, 1, 8), (256, 16, 8), (255, 3, 7)])
def test_against_the_block(e, n, topk):
    st = Stream()
    few = Few(layer(e), n, topk, st)
    x = synth.make_x(e + n, n, H)
    ref = reference(layer(e), x, topk)
    y = few.run(x)
    assert_rows(y, ref, range(n))
    for _ in range(3):  # the workspace is ready for the next call, and the same call gives the same bits
        assert np.array_equal(few.run(x), y)
    assert np.array_equal(few.run(x, in_place=True), y)
    assert device_error_word() == 0


@pytest.mark.parametrize("n,live", [(1, [0]), (2, [0, 1]), (5, [1, 0, 0, 1, 0]), (16, [0] * 15 + [1]), (16, [1, 0] * 8), (9, [0] * 9)])
def test_idle_rows_stay_as_they_were(n, live):
    st = Stream()
    few = Few(layer(16), n, 8, st)
    x = synth.make_x(3 * n, n, H)
    x[[i for i in range(n) if not live[i]]] = np.nan  # whatever an idle row holds
    ref = reference(layer(16), np.nan_to_num(x), 8)
    y = few.run(x, live)
    rows = [i for i in range(n) if live[i]]
    assert_rows(y, ref, rows)
    assert (y[[i for i in range(n) if not live[i]]] == 7.0).all()
    assert np.array_equal(few.run(x, live), y)
    assert device_error_word() == 0


def test_equal_logits_go_to_the_lower_index():
    host = dict(layer(64))
    host["moe.router"] = np.zeros_like(host["moe.router"])
    host["moe.router"][1::2] = synth.f32_to_bf16_bits(np.full((1, H), 2.0**-9, np.float32))  # the odd experts are equal, and so are the even ones
    st = Stream()
    few = Few(host, 3, 6, st)
    x = np.abs(synth.make_x(9, 3, H))
    x[1] = -x[1]  # the even experts' turn
    y = few.run(x)
    assert_rows(y, reference(host, x, 6), range(3))
    assert device_error_word() == 0


def test_rows_of_zeros_outliers_and_small_values():
    st = Stream()
    few = Few(layer(16), 6, 8, st)
    x = synth.make_x(4, 6, H)
    x[0] = 0
    x[1, 100] = 3e4       # one input far above its neighbours
    x[2] *= 1e-12         # eps rules the norm
    x[3] *= 1e10
    x[4, :64] = 0         # a group without a value
    y = few.run(x)
    ref = reference(layer(16), x, 8)
    # the outlier sets the digits of its 63 neighbours: 2^-24 of it each, which carries the row's norm, through at most eight sums
    assert np.array_equal(y[0], np.zeros(H, np.float32))
    assert np.linalg.norm(y[1] - ref[1]) <= (REL + 8 * 64**0.5 * 2.0**-24) * np.linalg.norm(ref[1])
    assert_rows(y, ref, (2, 3, 4, 5))
    assert device_error_word() == 0


@pytest.mark.parametrize("n", [3, 16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_row_that_is_not_finite_touches_no_other(n, bad):
    st = Stream()
    few = Few(layer(64), n, 8, st)
    x = synth.make_x(77, n, H)
    x[1, 1234] = bad
    live = [r != 1 for r in range(n)]
    want = few.run(np.nan_to_num(x), live)
    y = few.run(x)
    assert np.isnan(y[1]).all()
    ref = reference(layer(64), np.nan_to_num(x, posinf=0, neginf=0), 8)
    assert_rows(y, ref, [r for r in range(n) if r != 1])
    assert_rows(want, ref, [r for r in range(n) if r != 1])
    assert device_error_word() == 0


def test_one_workspace_serves_smaller_calls_and_other_layers():
    st = Stream()
    a = Few(layer(64), 16, 8, st)
    x = synth.make_x(31, 16, H)
    ya = a.run(x)
    for n, topk in ((1, 1), (16, 8), (5, 3), (9, 8)):
        y = a.run(x[:n], topk=topk)
        assert_rows(y, reference(layer(64), x[:n], topk), range(n))
    assert np.array_equal(a.run(x), ya)
    b = Few(layer(16), 16, 8, st)
    b.ws = a.ws
    assert_rows(b.run(x), reference(layer(16), x, 8), range(16))
    assert device_error_word() == 0


def test_replays_are_the_same_bits():
    st = Stream()
    few = Few(layer(64), 7, 8, st)
    x = synth.make_x(2, 7, H)
    y = few.run(x)
    dx, dy = DevBuf.from_array(x, st), DevBuf(7 * H * 4)
    g = Graph(st, lambda: [launched(few.call(dx, dy), "moe_few") for _ in range(3)])
    for _ in range(20):
        g.launch(st)
    assert np.array_equal(dy.download(np.float32, 7 * H, st).reshape(7, H), y)
    assert device_error_word() == 0


def test_two_calls_at_once():
    """Two streams, a workspace each: every launch gets the whole device, one after the other."""
    sts = [Stream(), Stream()]
    few = [Few(layer(e), n, 8, st) for e, n, st in zip((64, 16), (3, 16), sts)]
    xs = [synth.make_x(50 + f.n, f.n, H) for f in few]
    want = [f.run(x) for f, x in zip(few, xs)]
    dx = [DevBuf.from_array(x, st) for x, st in zip(xs, sts)]
    dy = [DevBuf.zeros(x.nbytes, st) for x, st in zip(xs, sts)]
    for st in sts:
        st.sync()
    for _ in range(30):
        for f, x, y in zip(few, dx, dy):
            launched(f.call(x, y), "moe_few")
    for f, y, w, st in zip(few, dy, want, sts):
        assert np.array_equal(y.download(np.float32, w.size, st).reshape(w.shape), w)
    assert device_error_word() == 0


def test_an_output_of_any_alignment():
    st = Stream()
    few = Few(layer(16), 5, 8, st)
    x = synth.make_x(3, 5, H)
    y = few.run(x)
    dx, out = DevBuf.from_array(x, st), DevBuf.zeros(5 * H * 4 + 16, st)
    w, live = few.w, None
    launched(few.l.drb_moe_few(C.byref(w), dx.at(0), out.at(4), live, 5, 16, 8, H, I, EPS, few.ws.at(0), st.raw), "moe_few")
    z = out.download(np.float32, 5 * H + 4, st)
    assert np.array_equal(z[1 : 5 * H + 1].reshape(5, H), y) and z[0] == 0 and (z[5 * H + 1 :] == 0).all()
