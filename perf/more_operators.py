"""The work a program hands to this library's passes in 8-bit floating point and to its log probabilities, as measurable cases.

  op        what is called                                                          stands for
  rows_f8   Runtime.rows_f8: rows normalised (after the residual's addition) or     the activations of a pass's projections, in e4m3 with a
            gated (silu(x) * x2), as e4m3 with a scale for each 128 columns         scale per token and 128 columns
  qmm_f8    Runtime.qmm_f8: such activations times an e4m3 weight tensor with a     projections of a decode step, a verification pass, a prompt
            scale for each block of 128 x 128
  logprobs  Runtime.logprobs: log probabilities of given tokens, entropies, top     scoring a prompt, the log probabilities that go with an answer
            alternatives

`run` computes them in elementary torch operations where `own` is false, and calls the library where it is true.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16}
F8 = torch.float8_e4m3fn
F8_MOST = 448.0
BLOCK = 128
EPS = 1e-6
MOST_BYTES = 6.3e8    # a drawn case's inputs and outputs, at most
MOST_MACS = 4096 * 17408 * 5120


def listed():
    return [
        # One decode step's row of hidden values: residual, norm, 8 bits.  Latency.
        {"name": "f8_rows_1", "op": "rows_f8", "ntok": 1, "cols": 5120, "type": "fp32", "residual": True, "norm": True, "gated": False},
        # A batch's verification passes: silu(gate) * up for the down projection, an odd number of rows.
        {"name": "f8_rows_gated", "op": "rows_f8", "ntok": 77, "cols": 17408, "type": "fp32", "residual": False, "norm": False, "gated": True},
        # A prompt pass, residual rows in 16 bits, a number of rows that is no multiple of anything.
        {"name": "f8_rows_prompt", "op": "rows_f8", "ntok": 4001, "cols": 5120, "type": "fp16", "residual": True, "norm": True, "gated": False},
        # The gate projection of a decode step: one pass over the weights.
        {"name": "f8_1", "op": "qmm_f8", "ntok": 1, "rows": 17408, "cols": 5120, "type": "fp32"},
        # A small projection of a verification pass: hardly anything to read.
        {"name": "f8_4_small", "op": "qmm_f8", "ntok": 4, "rows": 1024, "cols": 5120, "type": "fp32"},
        # The down projection of a batch's verification passes.
        {"name": "f8_24_down", "op": "qmm_f8", "ntok": 24, "rows": 5120, "cols": 17408, "type": "fp32"},
        # Odd sizes everywhere, blocks that end inside of 128.
        {"name": "f8_odd", "op": "qmm_f8", "ntok": 177, "rows": 1001, "cols": 4999, "type": "fp16"},
        # A prompt's chunk.
        {"name": "f8_512", "op": "qmm_f8", "ntok": 512, "rows": 17408, "cols": 5120, "type": "fp32"},
        # A long prompt, outputs in 16 bits.
        {"name": "f8_4096", "op": "qmm_f8", "ntok": 4096, "rows": 17408, "cols": 5120, "type": "fp16"},
        # The token that one sequence has just sampled, with twenty alternatives.  Latency.
        {"name": "logprobs_1", "op": "logprobs", "seqs": 1, "vocab": 151936, "type": "fp32", "top": 20, "temperature": False, "masked": False},
        # A batch with temperatures and a grammar's mask, an odd vocabulary.
        {"name": "logprobs_masked", "op": "logprobs", "seqs": 13, "vocab": 32003, "type": "fp32", "top": 5, "temperature": True, "masked": True},
        # Scoring a prompt.
        {"name": "logprobs_prompt", "op": "logprobs", "seqs": 2048, "vocab": 151936, "type": "fp16", "top": 1, "temperature": False, "masked": False},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["rows_f8", "qmm_f8", "qmm_f8", "logprobs"])
    kind = rng.choice(["fp32", "fp32", "fp16"])
    while True:
        if op == "rows_f8":
            gated = rng.random() < 0.35
            norm = not gated or rng.random() < 0.3
            case = {"op": op, "ntok": _log(rng, 1, 4096), "cols": _log(rng, 33, 20480), "type": kind, "residual": not gated and rng.random() < 0.7,
                    "norm": norm, "gated": gated}
        elif op == "qmm_f8":
            case = {"op": op, "ntok": _log(rng, 1, 4096), "rows": _log(rng, 17, 40000), "cols": _log(rng, 33, 20480), "type": kind}
            if case["ntok"] * case["rows"] * case["cols"] > MOST_MACS:
                continue
        else:
            case = {"op": op, "seqs": _log(rng, 1, 2048), "vocab": _log(rng, 101, 152064), "type": kind, "top": rng.randint(0, 20),
                    "temperature": rng.random() < 0.5, "masked": rng.random() < 0.3}
        if work(case)["bytes"] <= MOST_BYTES:
            return case


# ---- inputs ---------------------------------------------------------------------------------------------------------


class _State:
    """A pass's tensors, and where the library runs it the runtime that knows them by name."""

    def __init__(self, case, seed):
        self.case = case
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.t = {}
        self.rt = None
        if own:
            from vinf_3080ti_b200.runtime import Runtime

            self.rt = Runtime()

    def buffer(self, name, tensor):
        self.t[name] = tensor
        if self.rt is not None:
            self.rt.bind(name, tensor.data_ptr(), tensor.numel(), tensor.element_size())
        return tensor

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda")

    def uniform(self, low, high, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda") * (high - low) + low


def _up(n, to):
    return (n + to - 1) // to * to


def _padded(values, rows, cols):
    out = torch.zeros((rows, cols), dtype=values.dtype, device=values.device)
    out[:values.shape[0], :values.shape[1]] = values
    return out


def _quantised(blocks, dims):
    """(e4m3, scales) of values whose blocks lie along `dims`."""
    scale = (blocks.abs().amax(dims, keepdim=True).double() / F8_MOST).float()
    return torch.where(scale > 0, blocks.double() / scale.double(), 0.0).float().to(F8), scale


def prepare(case, seed):
    s = _State(case, seed)
    if case["op"] == "rows_f8":
        m, n, kind = case["ntok"], case["cols"], TYPES[case["type"]]
        channels = torch.where(s.uniform(0, 1, n) < 0.002, 20.0, 1.0)  # a few columns are much larger, as in hidden states
        s.buffer("x", (s.normal(m, n) * channels).to(kind))
        if case["gated"]:
            s.buffer("x2", s.normal(m, n).to(kind))
        if case["residual"]:
            s.buffer("residual", (s.normal(m, n) * 3 * channels).to(kind))
            s.buffer("sum", torch.zeros((m, n), dtype=kind, device="cuda"))
        if case["norm"]:
            s.buffer("gain", s.uniform(0.5, 1.5, n))
        s.buffer("q", torch.zeros((m, _up(n, 16)), dtype=torch.int8, device="cuda"))
        s.buffer("scale", torch.zeros((_up(n, BLOCK) // BLOCK, _up(m, 4)), device="cuda"))
    elif case["op"] == "qmm_f8":
        m, rows, cols, kind = case["ntok"], case["rows"], case["cols"], TYPES[case["type"]]
        kb, rb = _up(cols, BLOCK) // BLOCK, _up(rows, BLOCK) // BLOCK
        w = _padded(s.normal(rows, cols) * 0.02 * s.uniform(0.5, 2.0, rows, 1), rb * BLOCK, kb * BLOCK)
        w, w_scale = _quantised(w.view(rb, BLOCK, kb, BLOCK), (1, 3))
        # (kept as bytes, which is what the library's buffers hold; the rows lie on a grid of 16)
        s.t["w"] = w.view(rb * BLOCK, kb * BLOCK).view(torch.int8)[:rows, :_up(cols, 16)].contiguous()
        s.t["w_scale"] = w_scale.view(rb, kb).contiguous()
        del w
        if s.rt is not None:
            s.rt.bind_f8("w", s.t["w"].data_ptr(), s.t["w_scale"].data_ptr(), cols, rows)
        channels = torch.where(s.uniform(0, 1, cols) < 0.002, 20.0, 1.0)
        x, x_scale = _quantised(_padded(s.normal(m, cols) * channels, m, kb * BLOCK).view(m, kb, BLOCK), 2)
        s.buffer("q", x.view(m, kb * BLOCK).view(torch.int8)[:, :_up(cols, 16)].contiguous())
        s.buffer("scale", _padded(x_scale.view(m, kb).T, kb, _up(m, 4)))
        s.buffer("y", torch.zeros((m, rows), dtype=kind, device="cuda"))
    else:
        n, vocab, kind, top = case["seqs"], case["vocab"], TYPES[case["type"]], case["top"]
        logits = s.normal(n, vocab) * 3
        if case["masked"]:
            # what a grammar leaves: a tenth of the tokens; every seventh row only two
            left = s.uniform(0, 1, n, vocab) < 0.1
            left[:, 0] = True
            left[::7] = False
            left[::7, vocab // 3] = left[::7, vocab - 1] = True
            logits = torch.where(left, logits, -math.inf)
        s.buffer("logits", logits.to(kind))
        # a token that is likely, as a sampled one is, or any
        likely = (logits + 3 * s.normal(n, vocab)).argmax(-1)
        s.buffer("tokens", likely.int())
        del logits
        if case["temperature"]:
            s.buffer("temperature", s.uniform(0.5, 1.2, n))
        for name in ("out", "entropy"):
            s.buffer(name, torch.zeros(n, device="cuda"))
        if top:
            s.buffer("top_ids", torch.zeros((n, top), dtype=torch.int32, device="cuda"))
            s.buffer("top_out", torch.zeros((n, top), device="cuda"))
    torch.cuda.synchronize()
    return s


# ---- passes ---------------------------------------------------------------------------------------------------------


def _rows_f8(case, t):
    m, n, x = case["ntok"], case["cols"], t["x"]
    total = None
    v = x.float()
    if case["gated"]:
        v = v / (1 + torch.exp(-v)) * t["x2"].float()
    if case["residual"]:
        total = (v + t["residual"].float()).to(x.dtype)
        v = total.float()
    if case["norm"]:
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * t["gain"]
    blocks = _padded(v, m, _up(n, BLOCK)).view(m, -1, BLOCK)
    q, scale = _quantised(blocks, 2)
    return {"q": q.view(m, -1)[:, :n], "scale": scale[..., 0].T, "sum": total}


def _qmm_f8(case, t):
    m, rows, cols = case["ntok"], case["rows"], case["cols"]
    x = t["q"].view(F8)[:, :cols].float() * t["scale"][:, :m].T.repeat_interleave(BLOCK, 1)[:, :cols]
    w = t["w"].view(F8)[:, :cols].float() * t["w_scale"].repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return {"y": (x @ w.T).to(TYPES[case["type"]])}


def _logprobs(case, t):
    logits, top = t["logits"].float(), case["top"]
    at = t["temperature"][:, None] if case["temperature"] else 1.0
    less = (logits - logits.amax(-1, keepdim=True)) / at
    weights = torch.exp(less)
    sums = weights.sum(-1, keepdim=True)
    logs = less - torch.log(sums)
    # a token that is masked adds nothing
    entropy = -(weights / sums * torch.where(weights > 0, logs, 0.0)).sum(-1)
    answer = {"out": logs.gather(1, t["tokens"].long()[:, None])[:, 0], "entropy": entropy}
    if top:
        best, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
        ids = torch.nn.functional.pad(ids[:, :top], (0, max(0, top - case["vocab"])))
        best = torch.nn.functional.pad(best[:, :top], (0, max(0, top - case["vocab"])), value=-math.inf)
        answer["top_ids"] = torch.where(best > -math.inf, ids, -1).int()
        answer["top_out"] = torch.where(best > -math.inf, logs.gather(1, ids), -math.inf)
    return answer


def run(s):
    case, rt = s.case, s.rt
    op = case["op"]
    if not own:
        return _rows_f8(case, s.t) if op == "rows_f8" else _qmm_f8(case, s.t) if op == "qmm_f8" else _logprobs(case, s.t)
    if op == "rows_f8":
        rt.rows_f8("x", "q", "scale", case["cols"], case["ntok"], residual="residual" if case["residual"] else None,
                   total="sum" if case["residual"] else None, norm="gain" if case["norm"] else None, eps=EPS, silu_mul="x2" if case["gated"] else None)
        return {"q": s.t["q"].view(F8)[:, :case["cols"]], "scale": s.t["scale"][:, :case["ntok"]], "sum": s.t.get("sum")}
    if op == "qmm_f8":
        rt.qmm_f8("w", "q", "scale", "y", case["ntok"])
        return {"y": s.t["y"]}
    top = case["top"]
    rt.logprobs("logits", "tokens", case["vocab"], case["seqs"], out="out", entropy="entropy", top=top, top_ids="top_ids" if top else None,
                top_out="top_out" if top else None, temperature="temperature" if case["temperature"] else None)
    answer = {"out": s.t["out"], "entropy": s.t["entropy"]}
    if top:
        answer["top_ids"], answer["top_out"] = s.t["top_ids"], s.t["top_out"]
    return answer


# ---- what a pass cannot do without, and what it gives in 64 bits -----------------------------------------------------


def work(case):
    elem = 2 if case["type"] == "fp16" else 4
    if case["op"] == "rows_f8":
        values = case["ntok"] * case["cols"]
        read = values * elem * (1 + case["residual"] + case["gated"]) + 4 * case["cols"] * case["norm"]
        scales = 4 * case["ntok"] * (_up(case["cols"], BLOCK) // BLOCK)
        return {"bytes": read + values * (1 + elem * case["residual"]) + scales, "flops": values * (4 + 4 * case["norm"] + 5 * case["gated"])}
    if case["op"] == "qmm_f8":
        m, rows, cols = case["ntok"], case["rows"], case["cols"]
        kb, rb = _up(cols, BLOCK) // BLOCK, _up(rows, BLOCK) // BLOCK
        return {"bytes": rows * cols + m * cols + 4 * kb * (rb + m) + m * rows * elem, "flops": 2 * m * rows * cols}
    n, vocab, top = case["seqs"], case["vocab"], case["top"]
    return {"bytes": n * vocab * elem + 4 * n * (3 + case["temperature"] + 2 * top), "flops": 6 * n * vocab}


def exact(case, seed):
    t = prepare(case, seed).t

    def rows_in_64(case, t):
        cols, out = case["cols"], {"q": [], "scale": [], "sum": []}
        for r in range(0, case["ntok"], 512):  # a few rows at a time
            v = t["x"][r:r + 512].to(torch.float64)
            if case["gated"]:
                v = v * torch.sigmoid(v) * t["x2"][r:r + 512].to(torch.float64)
            if case["residual"]:
                v = torch.add(v, t["residual"][r:r + 512].to(torch.float64)).to(t["x"].dtype).to(torch.float64)
                out["sum"].append(v.clone())
            if case["norm"]:
                norm = torch.linalg.vector_norm(v, dim=1) / math.sqrt(cols)
                v = v / torch.sqrt(norm * norm + EPS)[:, None] * t["gain"].to(torch.float64)
            held, q = [], []
            for c in range(0, cols, 128):
                part = v[:, c:c + 128]
                largest = torch.maximum(part.max(1).values, -part.min(1).values) / 448
                held.append(largest)
                # (before it is rounded to 8 bits)
                q.append(torch.nan_to_num(part / largest[:, None]))
            out["q"].append(torch.cat(q, 1))
            out["scale"].append(torch.stack(held))
        return {"q": torch.cat(out["q"]), "scale": torch.cat(out["scale"], 1), "sum": torch.cat(out["sum"]) if out["sum"] else None}

    def logs_in_64(case, t):
        n, top = case["seqs"], case["top"]
        out = {"out": [], "entropy": [], "top_ids": [], "top_out": []}
        for r in range(0, n, 128):
            x = t["logits"][r:r + 128].to(torch.float64)
            if case["temperature"]:
                x = x / t["temperature"][r:r + 128, None].to(torch.float64)
            logs = torch.log_softmax(x, 1)
            out["out"].append(logs[torch.arange(len(x), device=x.device), t["tokens"][r:r + 128].long()])
            out["entropy"].append(torch.special.entr(torch.exp(logs)).sum(1))
            # of the same logits the one in front comes first
            at = torch.argsort(t["logits"][r:r + 128], dim=1, descending=True, stable=True)[:, :top]
            some = torch.gather(logs, 1, at)
            gone = torch.isneginf(some)
            out["top_ids"].append(at.masked_fill(gone, -1).to(torch.int32))
            out["top_out"].append(some)
        return {name: torch.cat(parts) for name, parts in out.items() if top or not name.startswith("top")}

    if case["op"] == "rows_f8":
        return rows_in_64(case, t)
    if case["op"] == "logprobs":
        return logs_in_64(case, t)
    m, rows, cols, parts = case["ntok"], case["rows"], case["cols"], []
    x = t["q"].view(F8)[:, :cols].to(torch.float64)
    for c in range(0, cols, 128):
        x[:, c:c + 128] *= t["scale"][c // 128, :m].to(torch.float64)[:, None]
    for r in range(0, rows, 2048):  # a few weight rows at a time
        w = t["w"][r:r + 2048, :cols].view(F8).to(torch.float64)
        for b in range(0, len(w), 128):
            for c in range(0, cols, 128):
                w[b:b + 128, c:c + 128] *= t["w_scale"][(r + b) // 128, c // 128].to(torch.float64)
        parts.append(x @ w.T)
    return {"y": torch.cat(parts, 1)}
