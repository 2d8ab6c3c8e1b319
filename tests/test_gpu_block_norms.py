"""drb_block_norms against the definition in 64 bits.

Tolerance, in units of u = 2^-24 relative to the value each rounding meets: a sum of squares of up to 8192 positive terms is added
up over at most 32 terms a thread, 5 butterfly steps and 32 warps, so it is off by at most 70 u, its root by 35 u, rsqrt and the division by 6 u more;
sigmoid 8 u; four products. So the second term of x' is off by at most 64 u of its size, x' by that and two u of either term, and h by 64 u of
its size and by x's own error; then h's type rounds by half a step.
"""

import numpy as np
import pytest
import torch

from drama_rs_b200 import ffi
from drama_rs_b200.gpu import DevBuf, Stream, launched
from tests.helpers import device_error_word

pytestmark = pytest.mark.gpu
TYPES = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}
U = 2.0**-24
EPS = 1e-6


def dev(t, st, lead=0):
    """Uploads a tensor `lead` values behind the start of a buffer; returns (buffer, offset in bytes)."""
    if t is None:
        return None, 0
    raw = t.contiguous().view(torch.uint8 if t.element_size() == 1 else {2: torch.int16, 4: torch.int32}[t.element_size()]).numpy()
    pad = np.zeros(lead, raw.dtype)
    return DevBuf.from_array(np.concatenate([pad, raw.reshape(-1)]), st), lead * t.element_size()


def at(b):
    return b[0].at(b[1]) if b[0] is not None else None


def run(o, post, gate, scale, alpha, x, pre, h_type, lead=0, in_place=False):
    st = Stream()
    rows, d = x.shape
    bufs = {k: dev(v, st, lead) for k, v in dict(o=o, post=post, gate=gate, scale=scale, x=x, pre=pre).items()}
    out = bufs["x"] if in_place else dev(torch.full_like(x, 5.0), st, lead)
    hz = dev(torch.full((rows, d), 5.0, dtype=TYPES[h_type]), st, lead)
    o_type = {v: k for k, v in TYPES.items()}[o.dtype]
    launched(ffi.lib().drb_block_norms(at(bufs["o"]), o_type, at(bufs["post"]), at(bufs["gate"]), at(bufs["scale"]), alpha, at(bufs["x"]), at(out),
                                       at(bufs["pre"]), at(hz) if pre is not None else None, h_type, rows, d, EPS, st.raw), "block_norms")
    xo = out[0].download(np.float32, rows * d, st, out[1]).reshape(rows, d)
    raw = hz[0].download(np.int32 if h_type == 0 else np.int16, rows * d, st, hz[1])
    return torch.from_numpy(xo), torch.from_numpy(raw).view(TYPES[h_type]).view(rows, d)


def check(o, post, gate, scale, alpha, x, pre, h_type, **kw):
    got_x, got_h = run(o, post, gate, scale, alpha, x, pre, h_type, **kw)
    f8 = torch.float64
    alpha = float(np.float32(alpha))
    t = o.to(f8)
    if post is not None:
        t = t / torch.sqrt((t * t).mean(1, keepdim=True) + EPS) * post.to(f8)
    if scale is not None:
        t = t * scale.to(f8)
    if gate is not None:
        t = t * torch.sigmoid(gate.to(f8))[:, None]
    r = alpha * x.to(f8)
    ref = r + t
    err = 66 * U * t.abs() + 2 * U * r.abs()
    assert ((got_x.to(f8) - ref).abs() <= err + 1e-30).all()
    if pre is None:
        assert (got_h.float() == 5.0).all()
        return got_x, got_h
    inv = 1.0 / torch.sqrt((ref * ref).mean(1, keepdim=True) + EPS)
    h = ref * inv * pre.to(f8)
    dt = TYPES[h_type]
    # the error of x' also moves the norm: by at most its rms over the row's rms
    moved = (err * err).mean(1, keepdim=True).sqrt() * inv
    tol = (err * inv * pre.to(f8).abs() + h.abs() * (64 * U + moved)) * 1.01
    tol = tol + (h.abs() + tol) * torch.finfo(dt).eps / 2 + (2.0**-25 if dt == torch.float16 else 1e-30)
    assert ((got_h.to(f8) - h).abs() <= tol).all()
    return got_x, got_h


def inputs(seed, rows, d, o_type=0, post=True, gate=True, scale=True, pre=True):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g)
    return dict(o=rn(rows, d).to(TYPES[o_type]), post=1 + 0.1 * rn(d) if post else None, gate=rn(rows) if gate else None,
                scale=0.3 + 0.05 * rn(d) if scale else None, alpha=0.875, x=1.5 * rn(rows, d), pre=1 + 0.1 * rn(d) if pre else None)


@pytest.mark.parametrize("rows,d", [(1, 1), (1, 2048), (3, 2049), (17, 1501), (300, 2048), (2, 8192), (5, 8191), (2, 4104), (7, 24), (33, 512)])
@pytest.mark.parametrize("o_type,h_type", [(0, 0), (0, 2), (1, 1), (2, 2), (1, 0)])
def test_against_the_definition(rows, d, o_type, h_type):
    check(**inputs(rows + d, rows, d, o_type), h_type=h_type)


@pytest.mark.parametrize("keep", [(), ("post",), ("gate",), ("scale",), ("post", "scale"), ("pre",), ("post", "gate", "pre")])
@pytest.mark.parametrize("d", [2048, 777])
def test_parts_that_are_left_out(keep, d):
    check(**inputs(5, 4, d, 1, *[k in keep for k in ("post", "gate", "scale", "pre")]), h_type=1)


@pytest.mark.parametrize("d", [2048, 1001])
def test_any_alignment_of_a_value(d):
    """A buffer that starts one value behind a 16-byte boundary gives the same as an aligned one of the same width form."""
    i = inputs(9, 6, d, 1)
    check(**i, h_type=2, lead=1)


def test_in_place_and_independent_of_the_other_rows():
    i = inputs(12, 40, 2048, 0)
    x0, h0 = run(**i, h_type=1)
    x1, h1 = run(**i, h_type=1, in_place=True)
    assert torch.equal(x0, x1) and torch.equal(h0, h1)
    one = {k: (v[7:8] if k in ("o", "x", "gate") else v) for k, v in i.items()}
    x2, h2 = run(**one, h_type=1)
    assert torch.equal(x2[0], x0[7]) and torch.equal(h2[0], h0[7])


def test_zero_rows_large_values_and_a_nan():
    i = inputs(20, 4, 2048, 0, gate=False)
    i["o"][0] = 0
    i["x"][0] = 0            # a row of zeros: rsqrt(eps) times zero
    i["o"][1] = 1e15         # squares up to 1e30 stay in range
    i["x"][2, 5] = float("nan")
    i["x"][3] *= 1e7         # fp16 rows stay within range after their norm
    clean = {k: (v[[0, 1, 3]] if k in ("o", "x") else v) for k, v in i.items()}
    check(**clean, h_type=2)
    x, h = run(**i, h_type=2)
    assert (x[0] == 0).all() and (h[0] == 0).all()
    assert torch.isnan(h[2].float()).all() and torch.isnan(x[2]).sum() == 1
    assert not torch.isnan(x[[0, 1, 3]]).any() and not torch.isnan(h[[0, 1, 3]].float()).any()


def test_fp16_rows_are_clamped():
    i = inputs(21, 1, 512, 0)
    i["pre"] = torch.full((512,), 1e6)
    _, h = run(**i, h_type=2)
    assert h.float().abs().max() == 65504.0 and torch.isfinite(h.float()).all()


def test_offsets_past_32_bits():
    """300,000 rows of 8192 (9.8 GB of x): zeros, but for the last row, which comes out as it does alone."""
    rows, d = 300_000, 8192
    st, l = Stream(), ffi.lib()
    g = np.random.default_rng(5)
    x1, w = g.standard_normal(d).astype(np.float32), (1 + 0.1 * g.standard_normal(d)).astype(np.float32)
    o1 = (g.standard_normal(d).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)  # bf16
    x, o, h = DevBuf.zeros(rows * d * 4, st), DevBuf.zeros(rows * d * 2, st), DevBuf.zeros(rows * d * 2, st)
    dw = DevBuf.from_array(w, st)

    def row(r):
        x.upload(x1, st, r * d * 4)
        o.upload(o1, st, r * d * 2)

    def call(r0, count):
        launched(l.drb_block_norms(o.at(r0 * d * 2), 1, dw.at(0), None, None, 0.5, x.at(r0 * d * 4), x.at(r0 * d * 4), dw.at(0), h.at(r0 * d * 2), 1, count, d,
                                   1e-6, st.raw), "block_norms")

    def got(r):
        return x.download(np.float32, d, st, r * d * 4), h.download(np.uint16, d, st, r * d * 2)

    row(rows - 1)
    call(rows - 1, 1)
    want = got(rows - 1)
    row(rows - 1)
    call(0, rows)
    for a, b in zip(got(rows - 1), want):
        assert np.array_equal(a, b)
    assert not got(rows - 2)[0].any() and device_error_word() == 0
