"""The step of several requests that decode together, as timed cases: what lies around and inside one layer.

A case is a plain dict with an "op":

  moe    one whole MoE layer for 1 to 16 tokens, one row per request (`drb_moe_few`); idle rows of a padded batch are
         not computed and their outputs stay as they are
  lora   an int8 projection of all rows with each row's low-rank adapter beside it (`drb_proj_q8_lora`)
  norms  post-norm of a block's output, gate, scaled residual and the next block's pre-norm (`drb_block_norms`)

With `own` false `run` computes the same in elementary torch operations; with `own` true it makes the library's calls.
`exact` restates each operator's definition in 64 bits.
"""

from __future__ import annotations

import ctypes as C
import math

import torch

own = False

H, I = 2048, 512  # hidden size and expert width of the backbone
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": 0, "bf16": 1, "f16": 2}


def listed() -> list[dict]:
    return [
        # one request alone: launches, waits and hand-overs, hardly any bytes
        {"name": "moe_1", "op": "moe", "rows": 1, "live": 1, "experts": 256, "topk": 8, "zipf": 0.0},
        # a handful of requests: nearly every (row, expert) pair has its own expert
        {"name": "moe_5", "op": "moe", "rows": 5, "live": 5, "experts": 256, "topk": 8, "zipf": 0.0},
        # a batch captured for 16 rows of which 11 are in use, popular experts shared by several rows
        {"name": "moe_16_11", "op": "moe", "rows": 16, "live": 11, "experts": 256, "topk": 8, "zipf": 1.1},
        # the largest batch of this form
        {"name": "moe_16", "op": "moe", "rows": 16, "live": 16, "experts": 256, "topk": 8, "zipf": 0.0},
        # one request's out-projection with its adapter and the residual
        {"name": "lora_1", "op": "lora", "rows": 1, "n": 2048, "k": 4096, "adapters": 1, "rank": 16, "type": "bf16", "res": True, "prompt": False},
        # in-projection of an odd number of requests over a few adapters
        {"name": "lora_17", "op": "lora", "rows": 17, "n": 8192, "k": 2048, "adapters": 6, "rank": 16, "type": "bf16", "res": False, "prompt": False},
        # many requests, nearly every one with an adapter of its own
        {"name": "lora_64", "op": "lora", "rows": 64, "n": 4096, "k": 2048, "adapters": 64, "rank": 32, "type": "f16", "res": False, "prompt": False},
        # chunks of three prompts in one call, each a run of rows with its own adapter
        {"name": "lora_300", "op": "lora", "rows": 300, "n": 4096, "k": 2048, "adapters": 3, "rank": 64, "type": "bf16", "res": False, "prompt": True},
        # between two blocks of one request's step
        {"name": "norms_1", "op": "norms", "rows": 1, "d": 2048, "o": "f32", "h": "f16", "post": True, "gate": True, "scale": True},
        # the same over a prompt's chunk
        {"name": "norms_300", "op": "norms", "rows": 300, "d": 2048, "o": "f32", "h": "bf16", "post": True, "gate": False, "scale": True},
        # a width that no vector load divides
        {"name": "norms_odd", "op": "norms", "rows": 777, "d": 1501, "o": "bf16", "h": "bf16", "post": True, "gate": True, "scale": False},
        # a long prompt in one call
        {"name": "norms_8192", "op": "norms", "rows": 8192, "d": 2048, "o": "bf16", "h": "bf16", "post": True, "gate": True, "scale": True},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(("moe", "lora", "norms"))
    if op == "moe":
        rows, experts = rng.randint(1, 16), rng.choice((16, 40, 64, 128, 256))
        live = rows if rng.random() < 0.6 else rng.randint(1, rows)
        return {"op": op, "rows": rows, "live": live, "experts": experts, "topk": rng.choice((1, 2, 4, 6, 8, 8)), "zipf": rng.choice((0.0, 1.1))}
    if op == "lora":
        k = rng.choice((512, 1024, 2048, 2176, 4096))
        n = _log_int(rng, 257, 4096 * 2048 // k)
        rank = rng.choice((8, 16, 24, 32, 64))
        prompt = rng.random() < 0.4
        rows = _log_int(rng, 65, 300) if prompt else _log_int(rng, 1, 64)
        return {"op": op, "rows": rows, "n": n, "k": k, "adapters": rng.randint(1, 4) if prompt else rng.randint(1, 32), "rank": rank,
                "type": rng.choice(("bf16", "f16")), "res": rng.random() < 0.5, "prompt": prompt}
    d = rng.choice((512, 1000, 1501, 2048, 2049, 4096))
    return {"op": op, "rows": _log_int(rng, 1, 6000 * 2048 // max(d, 2048)), "d": d, "o": rng.choice(("f32", "bf16", "f16")),
            "h": rng.choice(("f32", "bf16", "f16")) if d <= 2048 else "bf16", "post": rng.random() < 0.8, "gate": rng.random() < 0.5,
            "scale": rng.random() < 0.5}


# ----------------------------------------------------------------------------- inputs


class _Draw:
    """Seeded device tensors in the library's layouts."""

    def __init__(self, seed: int) -> None:
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def randn(self, *shape: int) -> torch.Tensor:
        return torch.randn(shape, device="cuda", generator=self.g)

    def q8(self, n: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
        """int8 codes and one f16 scale per 128 inputs of a row."""
        q = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=self.g)
        return q, (self.randn(n, k // 128) * 0.005).abs().clamp_min(1e-4).half()

    def q4(self, e: int, n: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Two int4 codes a byte (low nibble = even input) and f16 (scale, min) per 64 inputs."""
        q = torch.randint(0, 256, (e, n, k // 2), dtype=torch.uint8, device="cuda", generator=self.g)
        s = (self.randn(e, n, k // 64) * 0.01).abs().clamp_min(1e-4).half()
        return q, torch.stack((s, (s.float() * -8.0 + self.randn(e, n, k // 64) * 0.002).half()), dim=-1).contiguous()


def _inputs(case: dict, seed: int) -> dict:
    d = _Draw(seed)
    if case["op"] == "moe":
        n, e = case["rows"], case["experts"]
        router = d.randn(e + 1, H) * 0.02
        x = d.randn(n, H).bfloat16().float()
        if case["zipf"]:
            # popular experts: a direction that all rows share, weighted by each expert's rank
            common = d.randn(H)
            rank = torch.randperm(e, device="cuda", generator=d.g) + 1.0
            x = (0.8 * x + 0.6 * common).bfloat16().float()
            router[:e] += (-case["zipf"] * 0.4 * rank.log()).unsqueeze(1) * common * (1.6 / H)
        out = {"x": x, "router": router.bfloat16(), "norm": 1.0 + d.randn(H) * 0.1}
        out["sgu"], out["sd"], out["gu"], out["dn"] = d.q8(2 * I, H), d.q8(H, I), d.q4(e, 2 * I, H), d.q4(e, H, I)
        order = torch.randperm(n, device="cuda", generator=d.g)
        live = torch.zeros(n, dtype=torch.uint8, device="cuda")
        live[order[: case["live"]]] = 1
        out["live"] = live if case["live"] < n else None
        return out
    if case["op"] == "lora":
        rows, n, k, rank, held = case["rows"], case["n"], case["k"], case["rank"], case["adapters"]
        out = {"x": d.randn(rows, k).to(TYPES[case["type"]]), "w": d.q8(n, k)}
        out["a"] = (d.randn(held, rank, k) / math.sqrt(k)).bfloat16()
        out["b"] = (d.randn(held, n, rank) * 0.2).bfloat16()
        out["scale"] = 0.5 + torch.rand(held, device="cuda", generator=d.g)
        if case["prompt"]:  # runs of rows, the last one without an adapter
            cut = torch.arange(rows, device="cuda") * (held + 1) // rows
            who = torch.where(cut < held, cut, torch.full_like(cut, -1))
        else:
            who = torch.randint(-1, held, (rows,), device="cuda", generator=d.g)
            if rows == held:  # one adapter for each request
                who = torch.randperm(rows, device="cuda", generator=d.g)
        out["who"] = who.int()
        out["res"] = d.randn(rows, n) if case["res"] else None
        return out
    rows, dim = case["rows"], case["d"]
    return {"o": (d.randn(rows, dim) * 0.7).to(TYPES[case["o"]]), "x": d.randn(rows, dim) * 1.5,
            "post": 1.0 + d.randn(dim) * 0.1 if case["post"] else None, "gate": d.randn(rows) if case["gate"] else None,
            "scale": 0.3 + d.randn(dim) * 0.05 if case["scale"] else None, "pre": 1.0 + d.randn(dim) * 0.1, "alpha": 0.875}


def _p(t) -> C.c_void_p:
    return C.c_void_p(t.data_ptr() if t is not None else 0)


def prepare(case: dict, seed: int):
    state = {"case": case, "in": _inputs(case, seed)}
    t = state["in"]
    if case["op"] == "moe":
        state["y"] = torch.zeros((case["rows"], H), device="cuda")
    elif case["op"] == "lora":
        state["y"] = torch.empty((case["rows"], case["n"]), device="cuda")
        state["v"] = torch.empty((case["rows"], case["rank"]), device="cuda")
    else:
        state["x_out"], state["h"] = torch.empty_like(t["x"]), torch.empty_like(t["x"], dtype=TYPES[case["h"]])
    if own:
        from drama_rs_b200 import ffi
        from drama_rs_b200.gpu import check

        state["lib"] = ffi.lib()
        check(state["lib"].drb_init(), "init")
        if case["op"] == "moe":
            w = (t["router"], t["norm"], *t["gu"], *t["dn"], *t["sgu"], *t["sd"])
            state["weights"] = ffi.MoeLayerPtrs(*[v.data_ptr() for v in w])
            state["ws"] = torch.zeros(state["lib"].drb_moe_few_workspace_bytes(case["rows"], case["topk"]), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return state


# ----------------------------------------------------------------------------- one pass


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from drama_rs_b200.gpu import launched

    case, t, l = state["case"], state["in"], state["lib"]
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    if case["op"] == "moe":
        launched(l.drb_moe_few(C.byref(state["weights"]), _p(t["x"]), _p(state["y"]), _p(t["live"]), case["rows"], case["experts"], case["topk"],
                               H, I, EPS, _p(state["ws"]), st), "moe_few")
        return state["y"]
    if case["op"] == "lora":
        launched(l.drb_proj_q8_lora(_p(t["w"][0]), _p(t["w"][1]), _p(t["x"]), CODE[case["type"]], _p(t["a"]), _p(t["b"]), _p(t["scale"]), _p(t["who"]),
                                    case["adapters"], case["rank"], _p(t["res"]), _p(state["y"]), _p(state["v"]), case["rows"], case["n"], case["k"],
                                    st), "proj_q8_lora")
        return state["y"]
    launched(l.drb_block_norms(_p(t["o"]), CODE[case["o"]], _p(t["post"]), _p(t["gate"]), _p(t["scale"]), t["alpha"], _p(t["x"]), _p(state["x_out"]),
                               _p(t["pre"]), _p(state["h"]), CODE[case["h"]], case["rows"], case["d"], EPS, st), "block_norms")
    return {"x": state["x_out"], "h": state["h"]}


def _rms(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    return x * (1.0 / ((x * x).mean(dim=-1, keepdim=True) + EPS).sqrt()) * w


def _sigmoid(x: torch.Tensor) -> torch.Tensor:
    return 1.0 / (1.0 + (-x).exp())


def _wide8(w) -> torch.Tensor:
    q, s = w
    return (q.float().view(*s.shape, 128) * s.float().unsqueeze(-1)).view(q.shape)


def _wide4(q: torch.Tensor, sm: torch.Tensor) -> torch.Tensor:
    codes = torch.stack((q & 15, q >> 4), dim=-1).flatten(-2).float()
    sm = sm.float()
    return (codes.view(*sm.shape[:-1], 64) * sm[..., :1] + sm[..., 1:]).view(codes.shape)


def _run_plain(state):
    case, t = state["case"], state["in"]
    if case["op"] == "moe":
        e, x = case["experts"], t["x"]
        xh = _rms(x, t["norm"])
        logits = xh @ t["router"].float().T
        # descending, equal logits by index
        top, idx = torch.sort(logits[:, :e], dim=1, descending=True, stable=True)
        top, idx = top[:, : case["topk"]], idx[:, : case["topk"]]
        w = (top - top[:, :1]).exp()
        w = w / w.sum(dim=1, keepdim=True)
        gu = xh @ _wide8(t["sgu"]).T
        sh = (gu[:, :I] * _sigmoid(gu[:, :I]) * gu[:, I:]) @ _wide8(t["sd"]).T
        y = x + _sigmoid(logits[:, e:]) * sh
        for k in range(case["topk"]):
            sel = idx[:, k]
            gu = (_wide4(t["gu"][0][sel], t["gu"][1][sel]) @ xh.unsqueeze(-1)).squeeze(-1)
            a = gu[:, :I] * _sigmoid(gu[:, :I]) * gu[:, I:]
            y = y + w[:, k : k + 1] * (_wide4(t["dn"][0][sel], t["dn"][1][sel]) @ a.unsqueeze(-1)).squeeze(-1)
        return y if t["live"] is None else torch.where(t["live"].bool().unsqueeze(1), y, state["y"])
    if case["op"] == "lora":
        x, who = t["x"].float(), t["who"].long()
        y = x @ _wide8(t["w"]).T
        if t["res"] is not None:
            y = y + t["res"]
        for j in range(case["adapters"]):
            mine = (who == j).unsqueeze(1)
            v = (x * mine) @ t["a"][j].float().T
            y = y + t["scale"][j] * (v @ t["b"][j].float().T)
        return y
    o, x = t["o"].float(), t["x"]
    if t["post"] is not None:
        o = _rms(o, t["post"])
    if t["scale"] is not None:
        o = o * t["scale"]
    if t["gate"] is not None:
        o = o * _sigmoid(t["gate"]).unsqueeze(1)
    x = t["alpha"] * x + o
    return {"x": x, "h": _rms(x, t["pre"]).to(TYPES[case["h"]])}


# ----------------------------------------------------------------------------- the definitions in 64 bits


def exact(case: dict, seed: int):
    t = _inputs(case, seed)
    f8 = torch.float64
    if case["op"] == "norms":
        o, x = t["o"].to(f8), t["x"].to(f8)
        if t["post"] is not None:
            o = t["post"].to(f8) * o / torch.sqrt((o**2).sum(1, keepdim=True) / case["d"] + EPS)
        factor = torch.ones_like(o)
        if t["scale"] is not None:
            factor = factor * t["scale"].to(f8)
        if t["gate"] is not None:
            factor = factor * torch.sigmoid(t["gate"].to(f8))[:, None]
        x = x * t["alpha"] + factor * o
        return {"x": x, "h": t["pre"].to(f8) * x / torch.sqrt((x**2).sum(1, keepdim=True) / case["d"] + EPS)}
    if case["op"] == "lora":
        x = t["x"].to(f8)
        q, s = t["w"]
        y = x @ (q.to(f8) * s.to(f8).repeat_interleave(128, dim=1)).T
        for r, j in enumerate(t["who"].tolist()):
            if j >= 0:
                y[r] += float(t["scale"][j]) * (t["b"][j].to(f8) @ (t["a"][j].to(f8) @ x[r]))
        return y if t["res"] is None else y + t["res"].to(f8)

    def q4(pair, j):
        low, high = (pair[0][j] & 15).to(f8), (pair[0][j] >> 4).to(f8)
        codes = torch.empty(low.shape[0], 2 * low.shape[1], dtype=f8, device="cuda")
        codes[:, 0::2], codes[:, 1::2] = low, high
        sm = pair[1][j].to(f8).repeat_interleave(64, dim=1)
        return codes * sm[..., 0] + sm[..., 1]

    def q8(pair):
        return pair[0].to(f8) * pair[1].to(f8).repeat_interleave(128, dim=1)

    def mlp(up, down, v):
        z = up @ v
        return down @ (torch.nn.functional.silu(z[:I]) * z[I:])

    y = torch.zeros((case["rows"], H), dtype=f8, device="cuda")
    shared = (q8(t["sgu"]), q8(t["sd"]))
    for r in range(case["rows"]):
        if t["live"] is not None and not bool(t["live"][r]):
            continue
        x = t["x"][r].to(f8)
        v = x / torch.sqrt((x * x).mean() + EPS) * t["norm"].to(f8)
        logits = (t["router"].to(f8) @ v).tolist()
        chosen = sorted(range(case["experts"]), key=lambda j: (-logits[j], j))[: case["topk"]]
        weight = [math.exp(logits[j] - logits[chosen[0]]) for j in chosen]
        y[r] = x + mlp(*shared, v) / (1.0 + math.exp(-logits[-1]))
        for j, wj in zip(chosen, weight):
            y[r] += wj / sum(weight) * mlp(q4(t["gu"], j), q4(t["dn"], j), v)
    return y


# ----------------------------------------------------------------------------- what a pass cannot do without


def work(case: dict) -> dict:
    if case["op"] == "moe":
        m, e, topk = case["live"], case["experts"], case["topk"]
        expert = 3 * H * I // 2 + 3 * H * I // 64 * 4
        # experts that independent uniform choices of the live rows reach (popular experts: somewhat fewer)
        hit = e * (1.0 - (1.0 - topk / e) ** m)
        return {"bytes": hit * expert + 3 * H * I * (1 + 2 / 128) + (e + 1) * H * 2 + 8 * m * H + 4 * H,
                "flops": 2.0 * m * ((e + 1) * H + (topk + 1) * 3 * H * I)}
    if case["op"] == "lora":
        rows, n, k, rank = case["rows"], case["n"], case["k"], case["rank"]
        hit = min(case["adapters"], rows)
        return {"bytes": n * k * (1 + 2 / 128) + hit * rank * (n + k) * 2 + rows * (2 * k + 4 * n * (2 if case["res"] else 1)),
                "flops": 2.0 * rows * (n * k + rank * (n + k))}
    size = {"f32": 4, "bf16": 2, "f16": 2}
    return {"bytes": case["rows"] * case["d"] * (8 + size[case["o"]] + size[case["h"]]), "flops": 12.0 * case["rows"] * case["d"]}
