"""Several requests decoding together: the batch decoder, and the three calls of a step behind one another, eager and replayed.

Tolerance of the whole step: every call by itself is held to a few units of 2^-24 (their own tests); the 16-bit rows between them round by half a
step of bf16, 2^-9 relative, and the reference here rounds the same values at the same places. A value next to a boundary may round the other
way, which is a whole step, 2^-8, of one input in some hundred: over sums of 2048 inputs 2^-8 / sqrt(100) / sqrt(2048) of a sum's typical size
for each, far below the 1e-4 allowed on a row's 2-norm.
"""

import numpy as np
import pytest

from drama_rs_b200 import synth
from drama_rs_b200.engine import MoeBatchDecoder, MoeDecoder, block_norms, project_rows
from drama_rs_b200.gpu import DevBuf, Graph, Stream
from drama_rs_b200.model import Adapters, MoeLayer, Q8
from oracle import moe_oracle as orc
from tests.helpers import device_error_word

pytestmark = pytest.mark.gpu
H, EPS = 2048, 1e-6


def layers(count, e=16):
    return [synth.make_layer(70 + i, synth.MoeShape(experts=e)) for i in range(count)]


@pytest.mark.parametrize("n", [1, 5, 16])
def test_batch_decoder_steps(n):
    st = Stream()
    host = layers(3)
    dev = [MoeLayer.upload(h, st) for h in host]
    dec = MoeBatchDecoder(dev, n, st=st)
    x = synth.make_x(n, n, H)
    ref = x.astype(np.float64)
    for h in host:
        ref = orc.moe_layer(h, ref, 8, EPS, np.float64)[0]
    dec.set_x(x)
    y = dec.step()
    for r in range(n):
        assert np.linalg.norm(y[r] - ref[r]) <= 1.2e-5 * np.linalg.norm(ref[r])  # three layers of 4e-6
    dec.capture()
    for _ in range(3):
        dec.set_x(x)
        assert np.array_equal(dec.step(), y)
    # a captured step serves any number of live rows
    live = np.zeros(n, np.uint8)
    live[n // 2] = 1
    dec.set_live(live)
    dec.set_x(x)
    z = dec.step()
    others = np.arange(n) != n // 2
    assert np.array_equal(z[others], x[others])
    assert np.linalg.norm(z[n // 2] - ref[n // 2]) <= 1.2e-5 * np.linalg.norm(ref[n // 2])
    # one request alone is what the batch-1 decoder computes
    one = MoeDecoder(dev, st=st)
    one.set_x(x[0])
    w = one.step_eager()
    assert np.linalg.norm(w - y[0]) <= 1e-4 * np.linalg.norm(w)
    assert device_error_word() == 0


def test_two_captured_steps_share_a_workspace():
    st = Stream()
    dev = [MoeLayer.upload(h, st) for h in layers(1)]
    a, b = MoeBatchDecoder(dev, 9, st=st), MoeBatchDecoder(dev, 4, st=st)
    b.ws = a.ws  # large enough for both
    xa, xb = synth.make_x(1, 9, H), synth.make_x(2, 4, H)
    a.capture(), b.capture()
    a.set_x(xa), b.set_x(xb)
    ya, yb = a.step(), b.step()
    for _ in range(5):
        b.set_x(xb)
        assert np.array_equal(b.step(), yb)
        a.set_x(xa)
        assert np.array_equal(a.step(), ya)
    assert device_error_word() == 0


def bf16(a):
    return synth.f32_to_bf16_bits(a.astype(np.float32))


@pytest.mark.parametrize("n", [1, 6, 16])
def test_a_step_of_all_three(n):
    """norm -> in-projection with adapters -> (a mixer: the first half of its outputs) -> out-projection with adapters and norms around it
    -> MoE layer -> norms."""
    st = Stream()
    rng = np.random.default_rng(n)
    wide, rank, held = 4096, 16, 3
    wi, si = synth.make_q8(1, wide, H)
    wo, so = synth.make_q8(2, H, H)
    ad = [tuple(rng.standard_normal(s, dtype=np.float32) * f for s, f in (((held, rank, k), k**-0.5), ((held, m, rank), 0.2))) for m, k in ((wide, H), (H, H))]
    scale = (0.5 + rng.random(held)).astype(np.float32)
    who = rng.integers(-1, held, n).astype(np.int32)
    w_in, w_post, w_pre, w_end = (1 + 0.1 * rng.standard_normal((4, H))).astype(np.float32)
    gate = rng.standard_normal(n).astype(np.float32)
    host = layers(1)[0]
    x0 = synth.make_x(5, n, H)

    f8 = np.float64
    back = synth.bf16_bits_to_f32
    proj = lambda rows, q, s, a, b: np.stack([orc.dequant_q8(q, s, f8) @ r + (scale[j] * (back(bf16(b[j])).astype(f8) @ (back(bf16(a[j])).astype(f8) @ r)) if j >= 0 else 0)
                                              for r, j in zip(rows, who)])
    h = back(bf16(orc.rmsnorm(x0.astype(f8), w_in, EPS, f8))).astype(f8)
    mixed = back(bf16(proj(h, wi, si, *ad[0])[:, :H])).astype(f8)
    o = proj(mixed, wo, so, *ad[1])
    x1 = 0.875 * x0.astype(f8) + (1 / (1 + np.exp(-gate.astype(f8))))[:, None] * orc.rmsnorm(o, w_post, EPS, f8)
    x2 = orc.moe_layer(host, x1, 8, EPS, f8)[0]
    end = orc.rmsnorm(x2, w_end, EPS, f8)

    up = lambda a: DevBuf.from_array(np.ascontiguousarray(a), st)
    qi, qo = Q8(up(wi), up(si), wide, H), Q8(up(wo), up(so), H, H)
    ai, ao = (Adapters.upload(bf16(a), bf16(b), scale, st) for a, b in ad)
    dwho, dgate, dnorm = up(who), up(gate), [up(w) for w in (w_in, w_post, w_pre, w_end)]
    x, h16, y1, m16, y2, v, out = DevBuf(n * H * 4), DevBuf(n * H * 2), DevBuf(n * wide * 4), DevBuf(n * H * 2), DevBuf(n * H * 4), DevBuf(n * rank * 4), DevBuf(n * H * 4)
    zero = DevBuf.zeros(n * H * 4, st)
    moe = MoeBatchDecoder([MoeLayer.upload(host, st)], n, st=st)

    def mixer():  # stands for the host's own work: the first half of every row, rounded to bf16, on the host
        rows = y1.download(np.float32, n * wide, st).reshape(n, wide)[:, :H]
        m16.upload(bf16(rows), st)

    def first():
        block_norms(zero, 0, x, x, n, H, st, pre_w=dnorm[0], h=h16, h_type=1)  # the pre-norm alone
        project_rows(qi, h16, 1, y1, n, st, ai, dwho, v)

    def second():
        project_rows(qo, m16, 1, y2, n, st, ao, dwho, v)
        block_norms(y2, 0, x, moe.x, n, H, st, post_w=dnorm[1], gate=dgate, alpha=0.875)
        moe.record_step()
        block_norms(zero, 0, moe.x, moe.x, n, H, st, pre_w=dnorm[3], h=out, h_type=0)

    def run(a, b):
        x.upload(x0, st)
        a()
        mixer()
        b()
        return out.download(np.float32, n * H, st).reshape(n, H)

    y = run(first, second)
    for r in range(n):
        assert np.linalg.norm(y[r] - end[r]) <= 1e-4 * np.linalg.norm(end[r]), r
    g1, g2 = Graph(st, first), Graph(st, second)
    for _ in range(3):
        assert np.array_equal(run(lambda: g1.launch(st), lambda: g2.launch(st)), y)
    assert device_error_word() == 0
