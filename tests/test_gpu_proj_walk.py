"""drb_proj_q8_lora where a block of the tcgen05 form goes through several weight tiles: random codes and scales in every tile, many calls, each equal
in bits to the first, and that one held to the definition in 64 bits.

Tolerance as in test_gpu_proj_lora.py: with u = 2^-23 an output meets k / 16 roundings inside the multiplications, 3 k / 128 at the scales and a dozen where
residual and adapter join, in quadrature, each at most u times the root of the summed squares; six standard deviations."""

import numpy as np
import pytest
import torch

from drama_rs_b200 import ffi
from drama_rs_b200.gpu import Stream, launched
from tests.helpers import device_error_word

pytestmark = pytest.mark.gpu
U = 2.0**-23
SMS, MAX_C, TILE = 148, 80, 128


def columns(rows):
    ny = -(-rows // MAX_C)
    return -(-(-(-rows // ny)) // 16) * 16


def takes_tcgen05(rows, n, k, adapters, rank):
    """The rule of proj_rows.cuh (`many`): the shapes below have to reach the form that they are here for."""
    nc = columns(rows)
    nt = 4 if rows > 24 else -(-rows // 8)
    passes, tiles = -(-rows // (8 * nt)), -(-n // TILE)
    waves = -(-tiles * -(-rows // nc) // SMS)
    most = min(adapters, nc) if rank else 0
    met = min(most, rows) if rows <= 64 else (most + 3) // 4
    few = 3500 * (1 + (passes - 1) // 32) + (210, 245, 355, 400)[nt - 1] * passes * (n * k // 1000) // 1000
    tc = 3000 + waves * (450 * (k // 128) + 1250 * met)
    if rank:
        few += 3000 + n * max(rows, 8) // 100
        tc += 2500
    return tc < few


def tiles_a_block(rows, n):
    return -(-n // TILE) / (SMS // -(-rows // columns(rows)))


class Case:
    def __init__(self, seed, rows, n, k, x_type, adapters=0, rank=0, who=None):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rn = lambda *s: torch.randn(s, device="cuda", generator=g)
        self.dims = (rows, n, k, adapters, rank, x_type)
        self.q = torch.randint(-128, 128, (n, k), dtype=torch.int8, device="cuda", generator=g)
        self.s = (rn(n, k // 128) * 0.005).abs().clamp_min(1e-4).half()
        self.x = rn(rows, k).to(torch.bfloat16 if x_type == 1 else torch.float16)
        self.res, self.y, self.st = rn(rows, n), torch.empty((rows, n), device="cuda"), Stream()
        self.a = self.b = self.scale = self.who = self.v = None
        if rank:
            self.a, self.b = (rn(adapters, rank, k) / k**0.5).bfloat16(), (rn(adapters, n, rank) * 0.3).bfloat16()
            self.scale = 0.5 + torch.rand(adapters, device="cuda", generator=g)
            self.who, self.v = torch.tensor(who, dtype=torch.int32, device="cuda"), torch.empty((rows, rank), device="cuda")

    def call(self):
        """One call on rows of outputs that hold NaNs before it."""
        rows, n, k, adapters, rank, x_type = self.dims
        p = lambda t: t.data_ptr() if t is not None else None
        self.y.fill_(float("nan"))
        torch.cuda.synchronize()
        launched(ffi.lib().drb_proj_q8_lora(p(self.q), p(self.s), p(self.x), x_type, p(self.a), p(self.b), p(self.scale), p(self.who), adapters, rank, p(self.res),
                                            p(self.y), p(self.v), rows, n, k, self.st.raw), "proj_q8_lora")
        self.st.sync()
        return self.y

    def check(self, y):
        rows, n, k, adapters, rank, _ = self.dims
        x = self.x.double()
        v = va = None
        if rank:
            j = self.who.long()
            on = ((j >= 0) & (j < adapters)).double()
            j = j.clamp(0, adapters - 1)
            a, s = self.a.double(), (self.scale.double()[j] * on)[:, None]
            v = s * torch.einsum("rok,rk->ro", a[j], x)
            va = s * torch.einsum("rok,rk->ro", a[j] ** 2, x**2).sqrt()
        for n0 in range(0, n, 4096):
            at = slice(n0, min(n0 + 4096, n))
            w = self.q[at].double() * self.s[at].double().repeat_interleave(128, dim=1)
            ref = x @ w.T + self.res[:, at].double()
            tol = (k / 16 + 3 * k / 128 + 12) ** 0.5 * U * ((x * x) @ (w * w).T).sqrt() + U * self.res[:, at].double().abs()
            if rank:
                b = self.b[:, at].double()
                for i in range(adapters):
                    mine = (self.who == i).nonzero().flatten()
                    ref[mine] += v[mine] @ b[i].T
                    tol[mine] += (k / 64 + rank + 8) ** 0.5 * U * ((va[mine] ** 2 + v[mine] ** 2) @ (b[i] ** 2).T).sqrt()
            off = (y[:, at].double() - ref).abs() - 6 * tol
            assert (off <= 0).all(), (n0, float(off.max()), int((off > 0).sum()))


def many_calls(c, calls):
    first = c.call().clone()
    c.check(first)
    wrong = [i for i in range(1, calls) if not torch.equal(c.call(), first)]
    assert not wrong, (len(wrong), wrong[:5])
    assert device_error_word() == 0


# three to four tiles a block, the last one with few rows of W (odd n); two passes over W with seven
ALONE = [(16, 60_001, 768), (80, 60_001, 768), (16, 75_700, 8192), (80, 57_000, 8192), (150, 57_003, 2048)]


@pytest.mark.parametrize("x_type", [1, 2])
@pytest.mark.parametrize("rows,n,k", ALONE)
def test_several_tiles_without_adapters(rows, n, k, x_type):
    assert takes_tcgen05(rows, n, k, 0, 0) and tiles_a_block(rows, n) > 3
    many_calls(Case(rows + n + k, rows, n, k, x_type), 100)


# With none, one, two and three different adapters among a tile's rows (an odd number of them hands every stage of the codes from one set of convert warps
# to the other at a tile's end), ranks from the smallest to the largest, rows of one adapter behind one another and mixed
BESIDE = [(16, 75_700, 768, 1, 8), (16, 75_700, 8192, 1, 16), (16, 75_700, 8192, 2, 64), (16, 75_700, 8192, 3, 24), (80, 60_001, 768, 1, 64),
          (80, 60_001, 768, 2, 16), (80, 60_001, 768, 3, 40), (80, 57_000, 8192, 1, 16), (80, 57_000, 8192, 2, 8), (80, 57_000, 8192, 3, 64),
          (150, 57_003, 2048, 3, 16), (300, 40_000, 1024, 9, 32),
          (100, 32_768, 2048, 64, 16), (81, 40_001, 640, 12, 8), (161, 40_001, 1024, 5, 24)]  # and rows that a pass's columns do not divide


@pytest.mark.parametrize("x_type", [1, 2])
@pytest.mark.parametrize("rows,n,k,adapters,rank", BESIDE)
def test_several_tiles_with_adapters(rows, n, k, adapters, rank, x_type):
    assert takes_tcgen05(rows, n, k, adapters, rank) and tiles_a_block(rows, n) > 3
    rng = np.random.default_rng(rows + n + k + rank)
    mixed = rng.integers(-1, adapters, rows).tolist()
    runs = sorted(mixed)  # neighbours of one adapter: many rows' tiles differ in how many they meet
    for who in ([-1] * rows, [0] * rows, mixed, runs):
        many_calls(Case(rows + n + k, rows, n, k, x_type, adapters, rank, who), 100)
