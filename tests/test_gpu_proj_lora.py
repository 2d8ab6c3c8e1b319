"""drb_proj_q8_lora against the definition in 64 bits.

Tolerance of an output, u = 2^-23 (a tensor-core sum may round towards zero): the products of 16-bit x and 8-bit codes are exact. A sum over k
inputs meets k / 16 roundings inside the multiplications, 3 k / 128 at the scales and a dozen where slices, residual and adapter join;
with independent signs they add up in quadrature, each at most u times a partial sum, whose typical size is that of the root of the summed
squares `mag`. The adapter adds sqrt(k / 64 + rank + 8) u of its own size. Six standard deviations are allowed.
"""

import numpy as np
import pytest
import torch

from drama_rs_b200 import ffi
from drama_rs_b200.gpu import DevBuf, Stream, launched
from tests.helpers import device_error_word

pytestmark = pytest.mark.gpu
U = 2.0**-23
F8 = torch.float64


def make(seed, rows, n, k, adapters, rank, x_type, who=None, extreme=False):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g)
    q = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int64).to(torch.int8)
    if extreme:
        q = torch.where(torch.rand(n, k, generator=g) < 0.5, torch.tensor(-128, dtype=torch.int8), torch.tensor(127, dtype=torch.int8))
    t = {"q": q, "s": (rn(n, k // 128) * 0.005).abs().clamp_min(1e-4).half(), "x": rn(rows, k).to(torch.bfloat16 if x_type == 1 else torch.float16),
         "a": (rn(max(adapters, 1), max(rank, 1), k) / k**0.5).bfloat16(), "b": (rn(max(adapters, 1), n, max(rank, 1)) * 0.3).bfloat16(),
         "scale": 0.5 + torch.rand(max(adapters, 1), generator=g), "res": rn(rows, n),
         "who": torch.randint(-1, max(adapters, 1), (rows,), generator=g).int() if who is None else torch.tensor(who, dtype=torch.int32)}
    t["dims"] = (rows, n, k, adapters, rank, x_type)
    return t


def up(t, st):
    if t.dtype in (torch.bfloat16, torch.float16):
        t = t.view(torch.int16)
    return DevBuf.from_array(t.contiguous().numpy(), st)


def run(t, res=True, alias=False, repeat=1):
    rows, n, k, adapters, rank, x_type = t["dims"]
    st, l = Stream(), ffi.lib()
    b = {name: up(t[name], st) for name in ("q", "s", "x", "a", "b", "scale", "who", "res")}
    y = b["res"] if alias else DevBuf.from_array(np.full((rows, n), 9.0, np.float32), st)
    v = DevBuf(rows * max(rank, 1) * 4)
    p = lambda name: b[name].at(0) if rank else None
    for _ in range(repeat):
        launched(l.drb_proj_q8_lora(b["q"].at(0), b["s"].at(0), b["x"].at(0), x_type, p("a"), p("b"), p("scale"), p("who"), adapters, rank,
                                    b["res"].at(0) if res else None, y.at(0), v.at(0) if rank else None, rows, n, k, st.raw), "proj_q8_lora")
    out = torch.from_numpy(y.download(np.float32, rows * n, st).reshape(rows, n))
    assert device_error_word() == 0
    return out


def check(t, y, res=True):
    rows, n, k, adapters, rank, _ = t["dims"]
    x = t["x"].to(F8)
    w = t["q"].to(F8) * t["s"].to(F8).repeat_interleave(128, dim=1)
    ref, mag = x @ w.T, ((x * x) @ (w * w).T).sqrt()
    tol = (k / 16 + 3 * k / 128 + 12) ** 0.5 * U * mag
    if rank:
        for r, j in enumerate(t["who"].tolist()):
            if 0 <= j < adapters:
                a, b, s = t["a"][j].to(F8), t["b"][j].to(F8), float(t["scale"][j])
                v = s * (a @ x[r])
                ref[r] += b @ v
                va = s * ((a * a) @ (x[r] * x[r])).sqrt()
                tol[r] += (k / 64 + rank + 8) ** 0.5 * U * ((b * b) @ (va * va + v * v)).sqrt()
    if res:
        ref, tol = ref + t["res"].to(F8), tol + U * t["res"].to(F8).abs()
    bad = (y.to(F8) - ref).abs() - 6 * tol
    assert (bad <= 0).all(), (float(bad.max()), float(((y.to(F8) - ref).abs() / tol).max()))


SHAPES = [(1, 2048, 4096, 1, 16), (1, 1, 128, 1, 8), (3, 17, 256, 2, 8), (8, 257, 2176, 5, 24), (9, 300, 512, 3, 64), (16, 128, 1024, 2, 16),
          (17, 1000, 2048, 4, 16), (32, 15, 640, 3, 8), (33, 2100, 1024, 7, 8), (64, 512, 2048, 64, 32), (65, 100, 8192, 2, 16), (5, 33, 8064, 2, 56),
          (130, 513, 384, 3, 40), (300, 256, 2048, 3, 64)]
# wide enough for the tcgen05 form, from one tile of 16 rows to two of 80, and more than 64 rows of too many adapters for it
SHAPES += [(10, 40000, 512, 1, 24), (24, 16400, 2048, 1, 16), (40, 8300, 2048, 2, 64), (60, 20000, 1024, 6, 8), (65, 9000, 640, 3, 40), (150, 5000, 2048, 2, 16),
           (81, 20000, 256, 70, 8)]


@pytest.mark.parametrize("x_type", [1, 2])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_definition(shape, x_type):
    t = make(sum(shape), *shape, x_type)
    y = run(t)
    check(t, y)
    assert torch.equal(run(t, alias=True), y)  # the residual in place
    check(t, run(t, res=False), res=False)


@pytest.mark.parametrize("rows,n", [(1, 200), (12, 200), (70, 200), (12, 30000), (70, 9000)])
@pytest.mark.parametrize("adapters,rank", [(0, 0), (0, 16), (3, 0)])
def test_the_projection_alone(rows, n, adapters, rank):
    t = make(rows, rows, n, 768, adapters, rank, 1, who=[0] * rows)
    check(t, run(t))


def test_rows_without_an_adapter_and_indices_out_of_range():
    who = [0, -1, 2, 3, -(2**31), 2**31 - 1, 1, 0, 1]
    t = make(4, 9, 96, 512, 3, 16, 2, who=who)
    check(t, run(t))


@pytest.mark.parametrize("x_type", [1, 2])
def test_extreme_codes(x_type):
    t = make(8, 20, 64, 2048, 1, 8, x_type, extreme=True)
    check(t, run(t))


def test_same_bits_every_time():
    t = make(3, 40, 1111, 2048, 4, 32, 1)
    y = run(t)
    for _ in range(3):
        assert torch.equal(run(t, repeat=5), y)


def test_a_row_of_nans_touches_no_other():
    t = make(6, 6, 64, 512, 2, 8, 1, who=[0, 1, 0, 1, 0, 1])
    y = run(t)
    t["x"][2, 17] = float("nan")
    z = run(t)
    assert torch.isnan(z[2]).all() and torch.equal(z[[0, 1, 3, 4, 5]], y[[0, 1, 3, 4, 5]])


@pytest.mark.parametrize("rows,n", [(6, 300), (40, 300), (70, 300), (170, 300), (33, 9000), (70, 9000), (170, 9000)])
def test_a_broken_adapter_stays_with_its_own_rows(rows, n):
    who = [r % 4 - 1 for r in range(rows)]
    t = make(rows, rows, n, 512, 3, 16, 1, who=who)
    y = run(t)
    t["b"][1, 7, 3] = float("nan")
    t["b"][1, 9, 4] = float("inf")
    t["a"][2, 5, 100] = float("nan")
    z = run(t)
    sound = [r for r in range(rows) if who[r] < 1]
    assert torch.equal(z[sound], y[sound])
    one = [r for r in range(rows) if who[r] == 1]
    kept = [c for c in range(n) if c not in (7, 9)]
    assert torch.isnan(z[one, 7]).all() and not torch.isfinite(z[one, 9]).any() and torch.equal(z[one][:, kept], y[one][:, kept])
    assert torch.isnan(z[[r for r in range(rows) if who[r] == 2]]).all()


@pytest.mark.parametrize("rows,n", [(20, 700), (90, 700), (90, 9000)])
def test_two_calls_at_once_and_a_replay(rows, n):
    """Two streams with scratch of their own; then one of them captured, behind itself, and replayed."""
    from drama_rs_b200.gpu import Graph

    l, sts = ffi.lib(), [Stream(), Stream()]
    ts = [make(40 + i, rows + 3 * i, n, 1024, 3, 16, 1 + i) for i in range(2)]
    ref = [run(t) for t in ts]
    bufs, ys, vs = [], [], []
    for t, st in zip(ts, sts):
        bufs.append({name: up(t[name], st) for name in ("q", "s", "x", "a", "b", "scale", "who", "res")})
        ys.append(DevBuf.zeros(t["dims"][0] * n * 4, st)), vs.append(DevBuf(t["dims"][0] * 16 * 4))

    def call(i):
        b, (m, *_) = bufs[i], ts[i]["dims"]
        launched(l.drb_proj_q8_lora(*(b[a].at(0) for a in ("q", "s", "x")), 1 + i, *(b[a].at(0) for a in ("a", "b", "scale", "who")), 3, 16, b["res"].at(0),
                                    ys[i].at(0), vs[i].at(0), m, n, 1024, sts[i].raw), "proj_q8_lora")

    def got(i):
        m = ts[i]["dims"][0]
        return torch.from_numpy(ys[i].download(np.float32, m * n, sts[i]).reshape(m, n))

    for _ in range(20):
        call(0), call(1)
    assert torch.equal(got(0), ref[0]) and torch.equal(got(1), ref[1])
    g = Graph(sts[0], lambda: (call(0), call(0)))
    ys[0].zero(sts[0])
    for _ in range(5):
        g.launch(sts[0]), call(1)
    assert torch.equal(got(0), ref[0]) and torch.equal(got(1), ref[1]) and device_error_word() == 0


def test_more_rows_than_a_grid_has_passes():
    """64 rows, over and over: every copy comes out as the first, and that one by the definition."""
    rows, times = 64, 34000
    t = make(1, rows, 3, 128, 1, 0, 1)
    ref = dict(t)
    st, l = Stream(), ffi.lib()
    x = up(t["x"].repeat(times, 1), st)
    q, s = up(t["q"], st), up(t["s"], st)
    y = DevBuf.zeros(rows * times * 3 * 4, st)
    launched(l.drb_proj_q8_lora(q.at(0), s.at(0), x.at(0), 1, None, None, None, None, 0, 0, None, y.at(0), None, rows * times, 3, 128, st.raw), "proj_q8_lora")
    out = torch.from_numpy(y.download(np.float32, rows * times * 3, st).reshape(times, rows, 3))
    check(ref, out[0], res=False)
    assert (out == out[0]).all() and device_error_word() == 0


@pytest.mark.parametrize("rows", [1, 70])
def test_offsets_past_32_bits(rows):
    """280,000 rows of W of 8192 inputs and 64 adapters: zeros, but for the last ones."""
    n, k, adapters, rank, last = 280_000, 8192, 64, 64, 40
    t = make(rows, rows, last, k, adapters, rank, 1, who=[adapters - 1 - (r % 2) * adapters for r in range(rows)])
    st, l = Stream(), ffi.lib()
    zeros = {"q": n * k, "s": n * (k // 128) * 2, "b": adapters * n * rank * 2}
    b = {name: DevBuf.zeros(size, st) for name, size in zeros.items()}
    bits = lambda a: (a.view(torch.int16) if a.dtype != torch.int8 else a).contiguous().numpy()
    b["q"].upload(bits(t["q"]), st, (n - last) * k)
    b["s"].upload(bits(t["s"]), st, (n - last) * (k // 128) * 2)
    b["b"].upload(bits(t["b"][adapters - 1]), st, (adapters * n - last) * rank * 2)
    b.update({name: up(t[name], st) for name in ("x", "a", "scale", "who")})
    y, v = DevBuf.zeros(rows * n * 4, st), DevBuf(rows * rank * 4)
    launched(l.drb_proj_q8_lora(*(b[a].at(0) for a in ("q", "s", "x")), 1, *(b[a].at(0) for a in ("a", "b", "scale", "who")), adapters, rank, None, y.at(0),
                                v.at(0), rows, n, k, st.raw), "proj_q8_lora")
    out = torch.from_numpy(y.download(np.float32, rows * n, st).reshape(rows, n))
    check(t, out[:, n - last :].contiguous(), res=False)
    assert (out[:, : n - last] == 0).all() and device_error_word() == 0
