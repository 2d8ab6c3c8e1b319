"""What the Python calls of the several-request step check before they launch: that every buffer holds what the kernels read and write (no GPU needed)."""

from __future__ import annotations

import ctypes as C
from types import SimpleNamespace

import pytest

from drama_rs_b200 import engine
from drama_rs_b200.model import Adapters, Q8

ROWS, N, K, COUNT, RANK, D = 5, 48, 256, 3, 16, 40


class Buf:
    def __init__(self, nbytes: int) -> None:
        self.nbytes = nbytes

    def at(self, offset: int) -> C.c_void_p:
        return C.c_void_p(4096 + offset)


@pytest.fixture
def calls(monkeypatch):
    made = []
    lib = SimpleNamespace(drb_proj_q8_lora=lambda *a: made.append("proj") or 0, drb_block_norms=lambda *a: made.append("norms") or 0)
    monkeypatch.setattr(engine.ffi, "lib", lambda: lib)
    monkeypatch.setattr(engine, "launched", lambda code, what: None)
    return made


ST = SimpleNamespace(raw=None)
PROJECTION = {"w.q": N * K, "w.s": N * 2 * 2, "x": ROWS * K * 2, "y": ROWS * N * 4, "res": ROWS * N * 4, "adapters.a": COUNT * RANK * K * 2,
              "adapters.b": COUNT * N * RANK * 2, "adapters.scale": COUNT * 4, "adapter_of": ROWS * 4, "v": ROWS * RANK * 4}
NORMS = {"o": ROWS * D * 2, "x": ROWS * D * 4, "x_out": ROWS * D * 4, "post_w": D * 4, "gate": ROWS * 4, "scale": D * 4, "pre_w": D * 4, "h": ROWS * D * 2}


def project(sizes, adapters=True):
    b = {k: Buf(v) for k, v in sizes.items()}
    held = Adapters(b["adapters.a"], b["adapters.b"], b["adapters.scale"], COUNT, RANK, N, K) if adapters else None
    engine.project_rows(Q8(b["w.q"], b["w.s"], N, K), b["x"], 1, b["y"], ROWS, ST, held, b["adapter_of"], b["v"], b["res"])


def norms(sizes, h_type=2, o_type=1):
    b = {k: Buf(v) for k, v in sizes.items()}
    engine.block_norms(b["o"], o_type, b["x"], b["x_out"], ROWS, D, ST, b["post_w"], b["gate"], b["scale"], 1.0, b["pre_w"], b["h"], h_type)


def test_buffers_of_the_very_size_are_taken(calls):
    project(PROJECTION)
    norms(NORMS)
    assert calls == ["proj", "norms"]


@pytest.mark.parametrize("short", sorted(PROJECTION))
def test_the_projection_refuses_a_short_buffer(calls, short):
    with pytest.raises(ValueError, match=short):
        project(PROJECTION | {short: PROJECTION[short] - 1})
    assert calls == []


@pytest.mark.parametrize("short", sorted(NORMS))
def test_the_norms_refuse_a_short_buffer(calls, short):
    with pytest.raises(ValueError, match=short):
        norms(NORMS | {short: NORMS[short] - 1})
    assert calls == []


def test_wider_types_need_wider_buffers(calls):
    for kw in (dict(h_type=0), dict(o_type=0)):
        with pytest.raises(ValueError):
            norms(NORMS, **kw)
    assert calls == []


def test_what_is_left_out_is_not_looked_at(calls):
    project(PROJECTION | {"adapter_of": 0, "v": 0}, adapters=False)
    b = {k: Buf(v) for k, v in NORMS.items()}
    engine.block_norms(b["o"], 1, b["x"], b["x_out"], ROWS, D, ST)
    engine.block_norms(b["o"], 1, b["x"], b["x_out"], ROWS, D, ST, h=Buf(0))
    assert calls == ["proj", "norms", "norms"]


def test_adapters_of_another_projection_are_refused(calls):
    b = {k: Buf(2 * v) for k, v in PROJECTION.items()}
    w = Q8(b["w.q"], b["w.s"], N, K)
    for n, k, of, v in ((N + 1, K, b["adapter_of"], b["v"]), (N, K + 128, b["adapter_of"], b["v"]), (N, K, None, b["v"]), (N, K, b["adapter_of"], None)):
        with pytest.raises(ValueError):
            engine.project_rows(w, b["x"], 1, b["y"], ROWS, ST, Adapters(b["adapters.a"], b["adapters.b"], b["adapters.scale"], COUNT, RANK, n, k), of, v)
    assert calls == []
