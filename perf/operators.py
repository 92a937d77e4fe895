"""Timed cases of the operators that serve a mixture of experts in 8-bit integers: routing by scores, residual + RMSNorm to 8-bit rows, the 8-bit
product with a scale for each token and channel, the SiLU gate to 8-bit rows, and one layer made of them.

`run` computes each in plain torch where `own` is false, and calls the library's device entries where it is true. Activations are N(0, 1), weights
8-bit codes of N(0, 1) / 30 with a scale for each channel, router logits N(0, 1) plus an offset for each expert, so that the load is uneven.
"""
import math

import torch

own = False
BF16 = torch.bfloat16
EPS = 1e-6
FLOOR = 2.0 ** -100                                 # least largest value of a row: a row of zeros has a scale too
MOST_NORM, MOST_GATE, MOST_GEMM = 4096 * 2048, 32768 * 768, 4096 * 4096 * 4096


def listed():
    return [
        # interactive decode: one token over many experts in groups, sigmoid scores and a balance bias
        {"name": "route_1", "kind": "route", "tokens": 1, "experts": 256, "topk": 8, "score": "sigmoid", "bias": True, "groups": 8, "kept": 4, "rank": 2, "norm": True, "bf16": False},
        # a decode batch over the experts of the benchmark's model
        {"name": "route_256", "kind": "route", "tokens": 256, "experts": 128, "topk": 8, "score": "softmax", "bias": False, "groups": 1, "kept": 1, "rank": 1, "norm": True, "bf16": True},
        # a long prefill over grouped experts
        {"name": "route_8192", "kind": "route", "tokens": 8192, "experts": 256, "topk": 8, "score": "sigmoid", "bias": True, "groups": 8, "kept": 4, "rank": 2, "norm": True, "bf16": False},
        # one token between two layers
        {"name": "norm_1", "kind": "norm", "tokens": 1, "hidden": 2048, "stream": "f32", "delta": "f32"},
        # a prefill chunk between two layers
        {"name": "norm_4096", "kind": "norm", "tokens": 4096, "hidden": 2048, "stream": "f32", "delta": "f32"},
        # a dense projection of one token: latency of a weight stream
        {"name": "gemm_1", "kind": "gemm", "m": 1, "n": 4096, "k": 4096, "out": "bf16"},
        # a ragged prefill chunk
        {"name": "gemm_300", "kind": "gemm", "m": 300, "n": 4096, "k": 2048, "out": "bf16"},
        # a long prefill
        {"name": "gemm_4096", "kind": "gemm", "m": 4096, "n": 4096, "k": 4096, "out": "bf16"},
        # the gate of a decode batch: 64 tokens x 8 picks
        {"name": "gate_512", "kind": "gate", "rows": 512, "inter": 768, "bf16": True},
        # the gate of a long prefill: 4096 tokens x 8 picks
        {"name": "gate_32768", "kind": "gate", "rows": 32768, "inter": 768, "bf16": True},
        # norm and expert layer of a decode batch
        {"name": "layer_64", "kind": "layer", "tokens": 64, "experts": 128, "topk": 8, "hidden": 2048, "inter": 768, "score": "sigmoid", "bias": True, "groups": 8, "kept": 4, "rank": 2},
        # norm and expert layer of a long prefill
        {"name": "layer_4096", "kind": "layer", "tokens": 4096, "experts": 128, "topk": 8, "hidden": 2048, "inter": 768, "score": "softmax", "bias": False, "groups": 1, "kept": 1, "rank": 1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _routing(rng, experts):
    groups = rng.choice([g for g in (1, 1, 4, 8) if experts % g == 0 and experts // g >= 4])
    kept = rng.randint(max(1, groups // 4), groups)
    topk = min(rng.choice((1, 2, 4, 6, 8)), kept * (experts // groups))
    return {"topk": topk, "score": rng.choice(("sigmoid", "softmax")), "bias": rng.random() < 0.5, "groups": groups, "kept": kept, "rank": rng.choice((1, 2))}


def draw(rng):
    kind = rng.choice(("route", "norm", "gemm", "gemm", "gate", "layer"))
    if kind == "route":
        experts = rng.choice((8, 60, 64, 100, 128, 160, 256, rng.randint(8, 256)))
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "experts": experts, "norm": rng.random() < 0.7, "bf16": rng.random() < 0.5, **_routing(rng, experts)}
    if kind == "norm":
        hidden = 16 * _log(rng, 16, 512)
        return {"kind": kind, "tokens": _log(rng, 1, min(8192, MOST_NORM // hidden)), "hidden": hidden, "stream": rng.choice(("f32", "bf16")), "delta": rng.choice(("f32", "bf16", "none"))}
    if kind == "gemm":
        n, k, m = _log(rng, 64, 8192), 16 * _log(rng, 4, 512), _log(rng, 1, 4096)
        return {"kind": kind, "m": max(1, min(m, MOST_GEMM // (n * k))), "n": n, "k": k, "out": rng.choice(("bf16", "f32"))}
    if kind == "gate":
        inter = 16 * _log(rng, 8, 256)
        return {"kind": kind, "rows": _log(rng, 1, MOST_GATE // inter // 2), "inter": inter, "bf16": rng.random() < 0.7}
    experts, hidden, inter = rng.choice((8, 32, 60, 64)), 16 * rng.randint(32, 128), 16 * rng.randint(16, 48)
    return {"kind": kind, "tokens": _log(rng, 1, 4096), "experts": experts, "hidden": hidden, "inter": inter, **_routing(rng, experts)}


# ---------------------------------------------------------------------------------------------- what a program has in hand before the call
def _codes(g, *shape):
    return (torch.randn(shape, generator=g, device="cuda") * 30).round_().clamp_(-127, 127).to(torch.int8)


def _scales(g, count, about):
    return (0.5 + torch.rand(count, generator=g, device="cuda")) * about


def _router(case, g):
    logits = torch.randn((case["tokens"], case["experts"]), generator=g, device="cuda") + 0.5 * torch.randn(case["experts"], generator=g, device="cuda")
    return {"logits": logits.to(BF16) if case.get("bf16", True) else logits,
            "bias": 0.1 * torch.randn(case["experts"], generator=g, device="cuda") if case["bias"] else None}


def _stream(case, g):
    """residual stream, what the layer before adds to it, and the norm's weight"""
    shape = (case["tokens"], case["hidden"])
    h, m = torch.randn(shape, generator=g, device="cuda"), 0.5 * torch.randn(shape, generator=g, device="cuda")
    return {"h": h.to(BF16) if case.get("stream") == "bf16" else h, "m": {"bf16": m.to(BF16), "none": None}.get(case.get("delta", "f32"), m),
            "norm": 1 + 0.1 * torch.randn(case["hidden"], generator=g, device="cuda")}


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    if kind == "route":
        return _router(case, g)
    if kind == "norm":
        return _stream(case, g)
    if kind == "gate":
        gu = torch.randn((case["rows"], 2 * case["inter"]), generator=g, device="cuda")
        return {"gu": gu.to(BF16) if case["bf16"] else gu}
    if kind == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"x": _codes(g, m, k), "xs": _scales(g, m, 0.03), "w": _codes(g, n, k), "ws": _scales(g, n, 0.02 / 30)}
    E, H, I = case["experts"], case["hidden"], case["inter"]
    return {**_stream(case, g), **_router(case, g), "gate_up": _codes(g, E, 2 * I, H), "gate_up_s": _scales(g, E * 2 * I, 0.02 / 30),
            "down": _codes(g, E, H, I), "down_s": _scales(g, E * H, 0.02 / 30)}


class State:
    """One case's inputs, and for the library's entries the outputs, the arguments and the handles, which go back to it with the state (last made first)."""

    def __init__(self, case, data):
        self.case, self.data, self.handles, self.out, self.calls = case, data, [], None, []

    def __del__(self):
        while self.handles:
            free, handle = self.handles.pop()
            free(handle)


def _ok(rc):
    if rc != 0:
        from cudapp_b200 import api
        raise RuntimeError("rc %d: %s" % (rc, api.last_error()))


def _config(case, api):
    return api.MoeRouteConfig(case["experts"], case["topk"], api.SCORE_SIGMOID if case["score"] == "sigmoid" else api.SCORE_SOFTMAX, case["groups"], case["kept"], case["rank"],
                              int(case.get("norm", True)), 1.0)


def _va(t):
    return 0 if t is None else t.data_ptr()


def _weights(state, api, w, scale):
    rc, handle = api.i8_upload_dev(w.numel() // w.shape[-1], w.shape[-1], _va(w), _va(scale))
    _ok(rc)
    state.handles.append((api.lib.omega_gpu_i8_free, handle))
    return handle


def _norm_call(state, api, stream):
    d, (T, H) = state.data, state.data["h"].shape
    d["new_h"], d["q"], d["s"] = torch.empty((T, H), device="cuda"), torch.empty((T, H), dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
    x16 = d["h"] if d["h"].dtype == BF16 else None
    state.calls.append((api.lib.omega_gpu_residual_norm_q8_async, (T, H, EPS, _va(x16), _va(d["m"]), int(d["m"] is not None and d["m"].dtype == BF16), 0 if x16 is not None else _va(d["h"]),
                                                                   _va(d["new_h"]), _va(d["norm"]), 0, _va(d["q"]), _va(d["s"]), stream)))


def _calls(state):
    """the arguments that a serving loop keeps: device addresses, handles, its stream"""
    from cudapp_b200 import api
    c, d, kind, stream = state.case, state.data, state.case["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "route":
        state.out = {"ids": torch.empty((c["tokens"], c["topk"]), dtype=torch.int32, device="cuda"), "weights": torch.empty((c["tokens"], c["topk"]), device="cuda")}
        state.calls.append((api.lib.omega_gpu_moe_route_async, (_config(c, api), c["tokens"], _va(d["logits"]), int(c["bf16"]), 0, _va(d["bias"]), _va(state.out["ids"]),
                                                                _va(state.out["weights"]), stream)))
    elif kind == "norm":
        _norm_call(state, api, stream)
        state.out = {"h": d["new_h"], "scale": d["s"], "x": torch.empty((c["tokens"], c["hidden"]), dtype=BF16, device="cuda")}
    elif kind == "gate":
        d["q"], d["s"] = torch.empty((c["rows"], c["inter"]), dtype=torch.int8, device="cuda"), torch.empty(c["rows"], device="cuda")
        state.calls.append((api.lib.omega_gpu_swiglu_q8_async, (c["rows"], c["inter"], _va(d["gu"]), int(c["bf16"]), _va(d["q"]), _va(d["s"]), stream)))
        state.out = {"scale": d["s"], "x": torch.empty((c["rows"], c["inter"]), dtype=BF16, device="cuda")}
    elif kind == "gemm":
        w = _weights(state, api, d.pop("w"), d["ws"])
        y = torch.empty((c["m"], c["n"]), dtype=BF16 if c["out"] == "bf16" else torch.float32, device="cuda")
        state.calls.append((api.lib.omega_gpu_i8_gemm_async, (w, c["m"], _va(d["x"]), 0, _va(d["xs"]), _va(y) if c["out"] == "bf16" else 0, _va(y) if c["out"] == "f32" else 0, stream)))
        state.out = {"y": y}
    else:
        gate_up, down = _weights(state, api, d.pop("gate_up"), d["gate_up_s"]), _weights(state, api, d.pop("down"), d["down_s"])
        rc, layer = api.moe_i8_layer_create(gate_up, down, _config(c, api), None if d["bias"] is None else d["bias"].cpu().numpy(), c["tokens"])
        _ok(rc)
        state.handles.append((api.lib.omega_gpu_moe_i8_layer_free, layer))
        _norm_call(state, api, stream)
        out = torch.empty((c["tokens"], c["hidden"]), dtype=BF16, device="cuda")
        state.calls.append((api.lib.omega_gpu_moe_i8_layer_q8_async, (layer, c["tokens"], _va(d["logits"]), _va(d["q"]), _va(d["s"]), 0, _va(out), stream)))
        state.out = {"h": d["new_h"], "out": out}


def prepare(case, seed):
    state = State(case, _inputs(case, seed))
    if own:
        _calls(state)
    return state


# ---------------------------------------------------------------------------------------------- the plain forms
def _route(c, logits, bias):
    """scores and selection in 64 bits up to the score's rounding, so that near ties fall the same way on every device"""
    l = logits.double()
    score = (1 / (1 + torch.exp(-l)) if c["score"] == "sigmoid" else torch.softmax(l, -1)).float()
    value = score if bias is None else score + bias
    if c["groups"] > 1 and c["kept"] < c["groups"]:
        by_group = value.view(len(value), c["groups"], -1)
        rank = by_group.sort(dim=-1, descending=True).values[..., :c["rank"]].sum(-1)
        kept = rank.sort(dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
        mask = torch.zeros_like(rank, dtype=torch.bool).scatter_(1, kept, True)
        value = torch.where(mask[..., None], by_group, -torch.inf).view(value.shape)
    ids = value.sort(dim=-1, descending=True, stable=True).indices[:, :c["topk"]]
    w = score.gather(1, ids)
    return ids, w / (w.sum(-1, keepdim=True) + 1e-20) if c.get("norm", True) else w


def _quant(y):
    s = y.abs().amax(-1).clamp(min=FLOOR) / 127
    return (y / s[:, None]).round().clamp(-127, 127), s


def _norm(d):
    h = d["h"].float() if d["m"] is None else d["h"].float() + d["m"].float()
    return h, *_quant(h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * d["norm"])


def _gate(gu):
    g, u = gu.float().chunk(2, -1)
    return _quant(g / (1 + torch.exp(-g)) * u)


def _layer(c, d):
    E, H, I, K, T = c["experts"], c["hidden"], c["inter"], c["topk"], c["tokens"]
    h, x, xs = _norm(d)
    ids, wts = _route(c, d["logits"], d["bias"])
    flat = ids.reshape(-1)
    order = flat.argsort(stable=True)                                 # picks by expert, token, slot
    expert, count = flat[order], torch.bincount(flat, minlength=E)
    place = torch.arange(T * K, device=flat.device) - (count.cumsum(0) - count)[expert]
    most = int(count.max())
    rows = x.new_zeros((E, most, H)).index_put_((expert, place), x[order // K])
    gu = torch.bmm(rows, d["gate_up"].float().transpose(1, 2))[expert, place] * (xs[order // K, None] * d["gate_up_s"].view(E, 2 * I)[expert])
    a, s = _gate(gu.to(BF16))
    rows = x.new_zeros((E, most, I)).index_put_((expert, place), a)
    y = torch.bmm(rows, d["down"].float().transpose(1, 2))[expert, place] * (s[:, None] * d["down_s"].view(E, H)[expert])
    picked = torch.empty_like(y).index_copy_(0, order, y.to(BF16).float()).view(T, K, H)
    return {"h": h, "out": (picked * wts[..., None]).sum(1).to(BF16)}


def _plain(c, d):
    if c["kind"] == "route":
        ids, w = _route(c, d["logits"], d["bias"])
        return {"ids": ids.int(), "weights": w}
    if c["kind"] == "norm":
        h, q, s = _norm(d)
        return {"h": h, "scale": s, "x": (q * s[:, None]).to(BF16)}
    if c["kind"] == "gate":
        q, s = _gate(d["gu"])
        return {"scale": s, "x": (q * s[:, None]).to(BF16)}
    if c["kind"] == "gemm":
        y = d["x"].float() @ d["w"].float().T * (d["xs"][:, None] * d["ws"])
        return {"y": y.to(BF16) if c["out"] == "bf16" else y}
    return _layer(c, d)


def run(state):
    if not own:
        return _plain(state.case, state.data)
    for entry, args in state.calls:
        rc = entry(*args)
        if rc:
            _ok(rc)
    if "x" in state.out:                                              # 8-bit rows are told as the values that they stand for
        torch.mul(state.data["q"], state.data["s"][:, None], out=state.out["x"])
    return state.out


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_route(c, logits, bias):
    l = logits.double()
    e = torch.exp(l - l.max(-1, keepdim=True).values)
    score = (torch.exp(l) / (torch.exp(l) + 1) if c["score"] == "sigmoid" else e / e.sum(-1, keepdim=True))
    value = score.float() + (0 if bias is None else bias)
    size = c["experts"] // c["groups"]
    for _ in range(c["groups"] - c["kept"]):                          # drop the group of least rank, the last one of equals, until as many as wanted are left
        rank = value.view(len(value), c["groups"], size).topk(c["rank"], -1).values.sum(-1)
        rank = torch.where(rank == -torch.inf, torch.inf, rank)
        least = c["groups"] - 1 - rank.flip(1).argmin(-1)
        value.view(len(value), c["groups"], size)[torch.arange(len(value)), least] = -torch.inf
    ids = []
    for _ in range(c["topk"]):
        best = (value == value.max(-1, keepdim=True).values).int().argmax(-1, keepdim=True)
        ids.append(best)
        value.scatter_(1, best, -torch.inf)
    ids = torch.cat(ids, 1)
    w = score.gather(1, ids)
    return ids, w / w.sum(-1, keepdim=True) if c.get("norm", True) else w


def _exact_quant(y):
    top = torch.maximum(y.max(-1).values, -y.min(-1).values)
    s = torch.where(top > FLOOR, top, FLOOR) / 127
    return torch.round(y / s.unsqueeze(1)), s


def _exact_norm(d):
    h = d["h"].double() + (0 if d["m"] is None else d["m"].double())
    return h, *_exact_quant(h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS) * d["norm"].double())


def _exact_gate(gu):
    half = gu.shape[1] // 2
    g, u = gu[:, :half].double(), gu[:, half:].double()
    return _exact_quant(g * u * torch.exp(-torch.log1p(torch.exp(-g))))


def exact(case, seed):
    c, d, kind = case, _inputs(case, seed), case["kind"]
    if kind == "route":
        return {"ids": None, "weights": _exact_route(c, d["logits"], d["bias"])[1]}
    if kind in ("norm", "gate"):
        h, (q, s) = None, (None, None)
        if kind == "norm":
            h, q, s = _exact_norm(d)
        else:
            q, s = _exact_gate(d["gu"])
        return {"scale": s, "x": q * s.unsqueeze(1), **({} if h is None else {"h": h})}
    if kind == "gemm":
        return {"y": torch.mm(d["x"].double(), d["w"].double().t()) * torch.outer(d["xs"].double(), d["ws"].double())}
    E, H, I = c["experts"], c["hidden"], c["inter"]
    h, x, xs = _exact_norm(d)
    ids, wts = _exact_route(c, d["logits"], d["bias"])
    out = torch.zeros((c["tokens"], H), dtype=torch.float64, device="cuda")
    for e in range(E):                                                # one expert after the other, its tokens only
        token, slot = (ids == e).nonzero(as_tuple=True)
        gu = torch.mm(x[token], d["gate_up"][e].double().t()) * torch.outer(xs[token], d["gate_up_s"][e * 2 * I:(e + 1) * 2 * I].double())
        a, s = _exact_gate(gu.to(BF16)) if len(token) else (gu[:, :I], gu[:, 0])
        y = torch.mm(a, d["down"][e].double().t()) * torch.outer(s, d["down_s"][e * H:(e + 1) * H].double())
        out.index_add_(0, token, y.to(BF16).double() * wts[token, slot].unsqueeze(1))
    return {"h": h, "out": out}


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def _distinct(experts, topk, tokens):
    """experts that `tokens` tokens with `topk` different picks each are expected to reach"""
    return experts * (1.0 - (1.0 - min(1.0, topk / experts)) ** tokens)


def work(case):
    c, kind = case, case["kind"]
    if kind == "route":
        T, E = c["tokens"], c["experts"]
        return {"bytes": T * E * (2 if c["bf16"] else 4) + 4 * E * int(c["bias"]) + 8 * T * c["topk"], "flops": 8.0 * T * E}
    if kind == "norm":
        each = {"f32": 4, "bf16": 2, "none": 0}
        return {"bytes": c["tokens"] * (c["hidden"] * (each[c["stream"]] + each[c["delta"]] + 4 + 1) + 4) + 4 * c["hidden"], "flops": 6.0 * c["tokens"] * c["hidden"]}
    if kind == "gate":
        return {"bytes": c["rows"] * (c["inter"] * ((4 if c["bf16"] else 8) + 1) + 4), "flops": 8.0 * c["rows"] * c["inter"]}
    if kind == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": n * k + m * k + 4 * (m + n) + m * n * (2 if c["out"] == "bf16" else 4), "flops": 2.0 * m * n * k}
    T, E, H, I = c["tokens"], c["experts"], c["hidden"], c["inter"]
    experts = _distinct(E, c["topk"], T) * (3 * H * I + 4 * (2 * I + H))
    return {"bytes": experts + 2 * T * E + T * H * (4 + 4 + 4 + 2), "flops": 6.0 * T * c["topk"] * H * I}
